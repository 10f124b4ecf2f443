/* C ABI of the operators a learned prior over a texture's symbols is made of, exported by libntc_hip.so:
 * token log probabilities with their gradient, an AdamW step over many tensors, matrix products in
 * 8-bit floating point with a power-of-two scale for each block of 128, and what a sequence model's blocks have beside them: layer norm,
 * rotary positions of several axes, and causal attention, with their gradients.
 *
 * Every pointer is a device pointer unless its comment says host; every launch goes to `stream` (a hipStream_t;
 * null is the default stream) of the current device, and no call waits, allocates or copies. A call returns 0, or
 * 1 with a reason in why[0..why_cap) when its arguments are refused (nothing is launched then), or 2 when the
 * runtime reports an error of the launch. Sizes of zero are no error: nothing is launched.
 */
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Where this library finds the runtime's hipStreamSynchronize: a program in which two HIP runtimes may be loaded compares it with its own. Streams,
 * and the order of work on them, are one runtime's; a stream of another is none that these calls can take. */
const void* ntc_op_runtime(void);

enum { NTC_F32 = 0, NTC_BF16 = 1, NTC_F16 = 2 };     /* element types */
enum { NTC_MAX_TOP = 32 };                           /* alternatives of ntc_op_token_logprobs */
enum { NTC_STATE_BLOCK = 256 };                      /* values that share one scale of an 8-bit optimizer state */

/* Log probabilities of given tokens. Rows are addressed in two levels: row r = outer * inner_rows + inner starts
 * at logits + outer * outer_stride + inner * inner_stride (elements), its V values are contiguous; its token is at
 * tokens[outer * token_outer_stride + inner * token_inner_stride], 32 or 64 bits wide. With y = x * inv_temperature:
 *   logprob = y_token - log sum exp y,  entropy = -sum p log p,  and the `top` largest y in descending order (equal
 * values by ascending index; NaN orders as -inf) as ids and log probabilities.
 * A token equal to ignore_index has logprob 0; another token outside [0, V) has logprob NaN. A row of only -inf has
 * logprob and top_logprob -inf and entropy 0; a NaN or +inf makes a row's results NaN.
 * stats (2 floats a row) is what the backward pass needs: the largest x (-inf for a row of only -inf) and the log2
 * of the sum of exp(y - its largest). workspace: ntc_op_token_logprobs_workspace() bytes of any contents, not shared by calls
 * that may overlap (null where that is 0). */
typedef struct ntc_logprobs_desc {
    const void* logits;
    const void* tokens;
    int64_t rows, inner_rows, V;
    int64_t outer_stride, inner_stride;
    int64_t token_outer_stride, token_inner_stride;
    int64_t ignore_index;
    int32_t dtype, token_bytes;
    int32_t top;
    float temperature;    /* from 2^-127 to 2^120 */
    float* logprob;       /* [rows] */
    float* entropy;       /* [rows] */
    float* stats;         /* [rows][2] */
    int64_t* top_ids;     /* [rows][top] */
    float* top_logprobs;  /* [rows][top] */
    void* workspace;
    /* backward only: gradients of the outputs (null: none), laid out as these are */
    const float* g_logprob;
    const float* g_entropy;
    const float* g_top;   /* [rows][top] */
    void* dlogits;        /* [rows][V], contiguous, of `dtype` */
} ntc_logprobs_desc;

size_t ntc_op_token_logprobs_workspace(int64_t rows, int64_t V, int32_t dtype, int32_t top);
int ntc_op_token_logprobs(const ntc_logprobs_desc* d, void* stream, char* why, size_t why_cap);
/* dlogits from logits, tokens, stats, entropy, top_ids and the gradients of the outputs:
 *   dx_v = 1/T [ g_lp (v == token) + sum_k g_top_k (v == id_k) - p_v (g_lp + sum_k g_top_k + g_H (log p_v + H)) ]
 * (g_lp counts as 0 where the token is ignored; rows of only -inf get 0). */
int ntc_op_token_logprobs_backward(const ntc_logprobs_desc* d, void* stream, char* why, size_t why_cap);

/* ---------------------------------------------------------------- AdamW
 * One step of AdamW over many tensors: with gradient g, step count c of the tensor (1 at its first step),
 *   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
 *   p = p (1 - lr weight_decay) - lr / (1 - b1^c) * m / (sqrt(v / (1 - b2^c)) + eps)
 * in 32-bit arithmetic, p rounded once to its type (the 32-bit copy in `master`, where there is one, is what is updated then).
 * The gradients' addresses, the rates that follow from the step counts, and `calls` are arguments of the launch: a captured graph repeats them.
 *
 * The state is flat: tensor i's values are at state_offset (a multiple of NTC_STATE_BLOCK) in exp_avg, exp_avg_sq and master;
 * the values between a tensor's end and the next multiple are 0. With state_bits 8 each block of 256 values has
 * an exponent byte E: m is a sign and an unsigned 4 + 3 bit float, v an unsigned 5 + 3 bit float (exponent, mantissa; the
 * largest exponent stands for [1, 2), exponent 0 for the multiples of an eighth of the smallest other power),
 * times 2^(E - 127). They are rounded stochastically: up with the probability of the part cut off, in units of 2^-16. The bits
 * are mix64(head + (position / 2) * phi) (the library's counter noise; head = mix64(seed ^ 5 << 56 ^ calls << 32)), 16 for m
 * and 16 for v, in the low half for even positions. v > 0 is not rounded to 0. A block with a value that is not
 * finite, or of 2^127 and more, has E = 255: all of its values read as NaN. */
typedef struct ntc_adamw_tensor {      /* one tensor, in device memory */
    void* param;
    int64_t numel, state_offset;
    int32_t param_type, first_chunk;   /* first_chunk: its first entry in chunk_tensor */
} ntc_adamw_tensor;

enum { NTC_ADAMW_CHUNK = 4096 };       /* values that one entry of chunk_tensor stands for */

typedef struct ntc_adamw_desc {
    const ntc_adamw_tensor* tensors;   /* [n], device */
    const int32_t* chunk_tensor;       /* device: the tensor of each chunk of 4096 values, tensors in order */
    const int64_t* first_chunk;        /* host [n + 1]: each tensor's first chunk, and their number */
    const void* const* grads;          /* host [n]: gradients (device), null: the tensor is left alone */
    const int32_t* grad_types;         /* host [n] */
    const int32_t* steps;              /* host [n]: c, this step included */
    int64_t n;
    void* exp_avg;                     /* float32, or uint8 with state_bits 8 */
    void* exp_avg_sq;
    uint8_t* exp_avg_exp;              /* state_bits 8: [values / 256] */
    uint8_t* exp_avg_sq_exp;
    float* master;                     /* or null */
    double lr, beta1, beta2, eps, weight_decay;
    uint64_t seed;
    uint32_t calls;                    /* which call this is: other random bits each time */
    int32_t state_bits;
} ntc_adamw_desc;

int ntc_op_adamw(const ntc_adamw_desc* d, void* stream, char* why, size_t why_cap);
/* The values that an 8-bit state stands for: count (a multiple of 256) values of m and of v as 32-bit floats. */
int ntc_op_adamw_moments(const void* exp_avg, const void* exp_avg_sq, const uint8_t* exp_avg_exp, const uint8_t* exp_avg_sq_exp,
                         int64_t count, float* m, float* v, void* stream, char* why, size_t why_cap);
/* The nearest 8-bit state to count (a multiple of 256) values of m and v (a v below 0, or -0, counts as 0). */
int ntc_op_adamw_encode(const float* m, const float* v, int64_t count, void* exp_avg, void* exp_avg_sq, uint8_t* exp_avg_exp,
                        uint8_t* exp_avg_sq_exp, void* stream, char* why, size_t why_cap);

/* ---------------------------------------------------------------- 8-bit floating point with a scale for each block of 128
 * A matrix [R][K] in 8 bits: codes (OCP e4m3: sign, 4 exponent bits, 3 mantissa bits, largest 448, no infinity), row-major with
 * rows of ntc_fp8_code_stride(K) bytes, K up to a multiple of 128, the rest 0; and one exponent byte E (the scale is
 * 2^(E - 127)) for each block of `block_rows` x 128 values, block_rows 1 or 128, row-major with rows of ntc_fp8_exp_stride(K)
 * bytes (the blocks of a row up to a multiple of 4, the rest 0). E is the smallest for which no finite value of the
 * block exceeds 448 scales (at least 0); values are rounded to nearest, ties to even. Infinities and NaN become NaN. */
#ifdef __cplusplus
#define NTC_CONST_FN static constexpr
#else
#define NTC_CONST_FN static inline
#endif
NTC_CONST_FN int64_t ntc_fp8_code_stride(int64_t K) { return (K + 127) / 128 * 128; }
NTC_CONST_FN int64_t ntc_fp8_exp_stride(int64_t K) { return (K + 511) / 512 * 4; }

/* x [R][K] (rows at row_stride elements, columns contiguous) to 8 bits: as it lies (codes, exps: blocks along K) and
 * transposed (codes_t [K][R], exps_t: blocks along R); either pair may be null. With block_rows 128 both hold the same values. */
typedef struct ntc_fp8_quantize_desc {
    const void* x;
    int64_t R, K, row_stride;
    int32_t dtype, block_rows;
    uint8_t *codes, *exps, *codes_t, *exps_t;
} ntc_fp8_quantize_desc;
int ntc_op_fp8_quantize(const ntc_fp8_quantize_desc* d, void* stream, char* why, size_t why_cap);
/* Two at once, a of block_rows 1 and b of block_rows 128 (a layer's values and its weights): one launch where their types agree. */
int ntc_op_fp8_quantize_pair(const ntc_fp8_quantize_desc* a, const ntc_fp8_quantize_desc* b, void* stream, char* why, size_t why_cap);

/* C [M][N] = A [M][K] B [N][K]^T over matrices in 8 bits, summed in 32 bits, rounded once to c_type; C's rows at ldc elements.
 * (The 8-bit matrix instruction adds eight neighbouring products at a time, each cut off 13 bits below the largest exponent among them - the sum of its
 * factors', a subnormal code's being 2^-6's -, and these sums in 32 bits: 1.5e-5 of a result's magnitude on random values, up to 7 * 2^-13 of each eight's
 * largest product, and up to 64 times that where its factors are subnormal codes, which are themselves good to a few bits. A 16-bit result's rounding
 * is above the first, and a 32-bit result holds no more.)
 * With a_type not NTC_FP8, A is a matrix of floats (rows at a_stride elements) that is taken to 8 bits on the way, in
 * blocks of 1 x 128: a_exps is not used then. K is at most 2^23. workspace: ntc_op_fp8_matmul_workspace() bytes. */
enum { NTC_FP8 = 3 };
typedef struct ntc_fp8_matmul_desc {
    const void* a;
    const uint8_t* a_exps;
    const uint8_t* b;
    const uint8_t* b_exps;
    void* c;
    void* workspace;
    int64_t M, N, K;
    int64_t a_stride, ldc;
    int32_t a_type, a_block_rows, b_block_rows, c_type;
} ntc_fp8_matmul_desc;
size_t ntc_op_fp8_matmul_workspace(int64_t M, int64_t N, int64_t K, int32_t a_type);
int ntc_op_fp8_matmul(const ntc_fp8_matmul_desc* d, void* stream, char* why, size_t why_cap);
/* The rows of A up to which it may be given as floats. */
int64_t ntc_op_fp8_matmul_float_rows(void);

/* ---------------------------------------------------------------- layer norm
 * Rows of C values, contiguous, at x_stride (dy_stride) elements; results are contiguous. With mean and variance (over C) of a row in 32 bits,
 *   h = (x - mean) / sqrt(variance + eps),  y = h weight + bias   (null: 1 and 0),
 * rounded once to x's type. weight and bias are of x's type or float32, both alike. stats (2 floats a row: mean and 1 / sqrt) is what the backward pass needs; null
 * where there is none. Backward, with t = dy weight:
 *   dx = (t - mean t - h mean(t h)) / sqrt(variance + eps),  dweight = sum over rows of dy h,  dbias = sum over rows of dy
 * (each may be null); the sums are 32-bit, in an order that depends on the sizes alone. A row with a value that is not finite is NaN.
 * workspace: ntc_op_layer_norm_workspace() bytes of any contents, for dweight and dbias. */
typedef struct ntc_layer_norm_desc {
    const void* x;
    const void* weight;
    const void* bias;
    void* y;
    float* stats;          /* [rows][2], at a multiple of 8 bytes */
    int64_t rows, C;
    int64_t x_stride, dy_stride;
    int32_t dtype, weight_type;
    float eps;
    /* backward only */
    const void* dy;
    void* dx;              /* [rows][C] */
    void* dweight;         /* [C], of weight_type */
    void* dbias;
    void* workspace;
} ntc_layer_norm_desc;
int ntc_op_layer_norm(const ntc_layer_norm_desc* d, void* stream, char* why, size_t why_cap);
size_t ntc_op_layer_norm_workspace(int64_t rows, int64_t C);
int ntc_op_layer_norm_backward(const ntc_layer_norm_desc* d, void* stream, char* why, size_t why_cap);

/* ---------------------------------------------------------------- rotary positions of several axes
 * Up to two tensors (queries and keys) of tokens x heads x head_dim elements, a head's contiguous, tokens and heads at any strides; results are
 * contiguous [tokens][heads][head_dim] and do not overlap what they are made from. A token has a position (an integer) on each of `axes` axes; axis m turns sections[m] pairs of a head's elements, in
 * order: pair p of all P is elements p and p + P, or with `interleaved` 2p and 2p + 1; elements from 2 P on stay as they are. The angle of an axis's pair j is its position times
 * base^(-j / sections[m]), or with one_ladder, of pair p, base^(-p / P). (a, b) becomes (a cos - b sin, a sin + b cos); with `backward` the
 * sine's sign is changed, which is the gradient. Frequencies are good to 2^-57 of them and angles are fractions of a turn in 64 bits: an angle is off by no more than its position times
 * (2^-57 of its frequency + 2^-65 of a turn). Sines, cosines and sums are 32-bit, rounded once. */
enum { NTC_ROTARY_AXES = 8, NTC_ROTARY_PAIRS = 128 };
typedef struct ntc_rotary_desc {
    const void* positions;                 /* [tokens] rows of `axes` integers, at position_stride elements */
    int64_t position_stride, tokens;
    const void* x[2];
    void* y[2];
    int64_t token_stride[2], head_stride[2];
    int32_t heads[2];                      /* 0: no such tensor; 2^28 elements a token at most */
    int32_t head_dim, axes, position_bytes, dtype, one_ladder, interleaved, backward;
    int32_t sections[NTC_ROTARY_AXES];
    double base;
} ntc_rotary_desc;
int ntc_op_rotary(const ntc_rotary_desc* d, void* stream, char* why, size_t why_cap);

/* ---------------------------------------------------------------- attention
 * Sequences of queries against keys and values, bfloat16 or float16, heads of head_dim elements (a multiple of 8, up to 128); q_heads is a
 * multiple of k_heads, and query head h reads key head h / (q_heads / k_heads). For query i and key j of a sequence of Lq and Lk,
 *   s = scale q_i k_j,  where causal: j <= i + Lk - Lq,  p = softmax over the keys that are left,  o_i = sum_j p_j v_j;
 * a query that has none left has o = 0 and lse = -inf. What the backward pass needs, null where there is none: lse (natural log sum exp s), [query rows][q_heads], and o_rest, what o's
 * rounding left (times 2^11 for float16), without which sum dO o is too coarse beside the differences dO v - D below.
 *
 * Rows: with cu_q (device, `sequences` + 1 ends, the first 0, ascending) sequence b's queries are rows cu_q[b] .. cu_q[b + 1] of q_rows; rows behind the last
 * sequence have o = 0 and no gradient. Without, each sequence has q_rows / sequences, in turn. Keys and values alike, with cu_k and k_rows. With
 * k_lens (device) a sequence has k_lens[b] keys, the first of those rows; the others are not read. Numbers that leave their rows are cut off at the rows' ends: wrong ones give wrong
 * results, and no access out of bounds. A row of q is at q_row_stride elements from the one before it, within a sequence and, with cu_q, from one sequence to the next; without, sequences are
 * at q_batch_stride. All starts and strides are multiples of 8 elements (16 bytes); rows are at most 2^22 apart, heads 2^20. o, dq, dk and dv are contiguous [rows][heads][head_dim].
 *
 * Scores, the softmax's maximum and sum and all sums of products are 32-bit; the probabilities, and backwards their gradients, are rounded to the operands' type for the products
 * that follow (float16: times 2^7, so that 2^-32 of a row's largest is half the smallest step; backwards the gradients
 * times a power of two that goes by a sequence's largest dO and v, for dq by the row's own dO). With D = sum dO o (o before its rounding), dS = p (dO v - D): dv = sum p dO, dq = scale sum dS k, dk = scale sum dS q, the last two over the group's heads.
 * A query that sees a key or value that is not finite is NaN where the formula is, and so is one all of whose scores are -inf (lse too; also where finite values' products leave 32 bits); any query of that sequence may
 * be as well (0 times infinity).
 * workspace: ntc_op_attention_workspace() bytes (backward 0 or 1), any contents, at a multiple of 16 bytes. */
typedef struct ntc_attention_desc {
    const void *q, *k, *v;
    void* o;
    void* o_rest;                          /* like o */
    float* lse;
    const int32_t *cu_q, *cu_k, *k_lens;
    int64_t sequences, q_rows, k_rows;
    int64_t q_row_stride, q_head_stride, q_batch_stride;
    int64_t k_row_stride, k_head_stride, k_batch_stride;
    int64_t v_row_stride, v_head_stride, v_batch_stride;
    int32_t q_heads, k_heads, head_dim, dtype, causal;
    float scale;                           /* above 0 */
    void* workspace;
    /* backward only */
    const void* d_o;                       /* rows and heads at the strides below */
    int64_t do_row_stride, do_head_stride, do_batch_stride;
    void *dq, *dk, *dv;                    /* null: not wanted */
} ntc_attention_desc;
size_t ntc_op_attention_workspace(const ntc_attention_desc* d, int32_t backward);
int ntc_op_attention(const ntc_attention_desc* d, void* stream, char* why, size_t why_cap);
int ntc_op_attention_backward(const ntc_attention_desc* d, void* stream, char* why, size_t why_cap);

#ifdef __cplusplus
}
#endif
