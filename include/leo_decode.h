/*
 * leo_decode.h -- C-ABI of the operators that take a model from activations to
 * its next symbol: matrix-vector products with 4-bit weights and group scales
 * (the readout of a served model), the control of logits (penalties for
 * repeated symbols, biases, grammar masks) and the draw of one symbol a row.
 *
 * Same manner as leo_hip.h: every call returns an int32 status (0 = ok) and
 * leo_hip_last_error() returns the message of the last failure on the calling
 * thread. All pointers inside the argument structs are device memory of the
 * device that `stream` (a hipStream_t; NULL = the default stream) belongs to,
 * which must be the calling thread's current device. Calls enqueue work on
 * `stream` and return without waiting; they allocate nothing, so they may be
 * captured into a HIP graph. Strides count elements; the last axis is dense.
 */
#ifndef LEO_DECODE_H
#define LEO_DECODE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations, logits and scales. */
enum { LEO_TYPE_F32 = 0, LEO_TYPE_F16 = 1, LEO_TYPE_BF16 = 2 };

/* A 4-bit weight matrix [outputs, inputs]:
 *     w[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])
 * with codes 0..15, `group` 32, 64 or 128, and zero = 8 where has_zeros is 0.
 * The last group of a row may be short. */
typedef struct LeoQ4Shape {
    uint64_t outputs;
    uint64_t inputs;
    uint32_t group;
    int32_t scale_type; /* LEO_TYPE_* */
    uint32_t has_zeros;
    uint32_t pad0;
} LeoQ4Shape;

/* Bytes of the device layout that leo_q4_layout writes. */
int32_t leo_q4_layout_bytes(const LeoQ4Shape* shape, uint64_t* bytes);

/* Lays a matrix out once for leo_q4_matvec. Row n of `codes` holds
 * ceil(inputs / 2) bytes, input 2j in the low half of byte j; codes_stride is
 * the bytes from row to row. scales [outputs, ceil(inputs / group)] of
 * scale_type and zeros (uint8 0..15, the same shape, NULL without zeros) have
 * their own row strides. `layout` (256-byte aligned) receives layout_bytes. */
typedef struct LeoQ4Source {
    LeoQ4Shape shape;
    const void* codes;
    int64_t codes_stride;
    const void* scales;
    int64_t scales_stride;
    const void* zeros;
    int64_t zeros_stride;
    void* layout;
    uint64_t layout_bytes;
} LeoQ4Source;
int32_t leo_q4_layout(const LeoQ4Source* source, void* stream);

/* y[m, n] = bias[n] + sum over k of x[m, k] * w[n, k] for `rows` rows of x.
 * Sums are held in 32 bits and rounded once to y_type. x enters its products in
 * half precision, float16 as it is, others under a power of two for each row and
 * 128 inputs: bfloat16 in one part, float in two (22 bits), both to 2^-39 of the
 * largest of those 128. Scales have to stay below 2^100 in magnitude: a group's sum
 * is scaled before that power of two is taken back. bias (float) may be NULL. y and
 * x share no memory. `workspace`: at least leo_q4_workspace_bytes()
 * bytes (none where that is 0), 256-byte aligned, whatever they hold; free again
 * when the call's work is done. */
typedef struct LeoQ4Product {
    LeoQ4Shape shape;
    const void* layout;
    uint64_t layout_bytes;
    uint64_t rows;
    const void* x;
    int64_t x_stride;
    const float* bias;
    void* y;
    int64_t y_stride;
    int32_t x_type;
    int32_t y_type;
    void* workspace;
    uint64_t workspace_bytes;
} LeoQ4Product;
int32_t leo_q4_workspace_bytes(const LeoQ4Shape* shape, uint64_t rows, int32_t x_type, uint64_t* bytes);
int32_t leo_q4_matvec(const LeoQ4Product* product, void* stream);

/* Control of logits [rows, symbols], in this order for each logit z of symbol v
 * that occurs c times in the row's history:
 *     c > 0:  z = (z > 0 ? z / repetition : z * repetition)
 *             z = z - (presence + frequency * c)
 *     z = z + the row's bias for v, if it lists one
 *     z = -inf where the row's mask bit for v is 0
 * Lists are ragged: row r owns entries offsets[r] .. offsets[r + 1] - 1.
 * History entries outside 0 .. symbols-1 are ignored, so are biases'; of several
 * biases for one symbol the row's last counts. repetition (> 0), presence and
 * frequency hold one float a row; NULL means 1, 0 and 0. masks holds mask_count
 * rows of ceil(symbols / 32) words, symbol v at bit v % 32 of word v / 32;
 * mask_rows chooses one for each row, -1 for none; any other number outside
 * 0 .. mask_count-1 allows nothing. Without mask_rows, row r uses mask r, or
 * mask 0 where mask_count is 1. out may be the logits themselves, but not overlap
 * them otherwise. */
typedef struct LeoLogitControl {
    uint64_t rows;
    uint64_t symbols;
    const void* logits;
    int64_t logits_stride;
    void* out;
    int64_t out_stride;
    int32_t type; /* of logits and out */
    uint32_t pad0;
    const int32_t* history;
    const int64_t* history_offsets; /* rows + 1, or NULL: no history */
    uint64_t history_count;         /* entries in history */
    const float* repetition;
    const float* presence;
    const float* frequency;
    const int32_t* bias_ids;
    const float* bias_values;
    const int64_t* bias_offsets; /* rows + 1, or NULL: no biases */
    uint64_t bias_count;
    const int32_t* masks; /* NULL: no masks; then mask_count is 0 and mask_rows NULL */
    int64_t masks_stride;
    uint64_t mask_count;
    const int32_t* mask_rows;
} LeoLogitControl;
int32_t leo_control_logits(const LeoLogitControl* control, void* stream);

/* One symbol a row of logits [rows, symbols]. With z = logit / temperature in
 * float (a finite logit's does not fall below the lowest finite value) and
 * w = exp(z - max z), a symbol stays if fewer than top_k symbols have a larger z,
 * those have less than top_p of the whole mass (top_p >= 1: any), and
 * w >= min_p; the largest always stays. The symbol is the one that stays with
 * the largest z + noise (Gumbel noise, one value a logit), the lowest of equals;
 * a temperature that is not above 0 takes the largest logit, without noise or
 * filters. out_logprobs receives z - log sum exp z over the whole row (at
 * temperature 0, of the logits). A NaN logit counts as -inf; a row of -inf alone
 * gives symbol -1 and -inf. temperature, top_k, top_p and min_p hold one value a
 * row; NULL means 1, `symbols`, 1 and 0. noise NULL: every row takes its largest
 * logit, as at temperature 0. `workspace` as in leo_q4_matvec. */
typedef struct LeoSample {
    uint64_t rows;
    uint64_t symbols;
    const void* logits;
    int64_t logits_stride;
    int32_t type;
    uint32_t pad0;
    const float* noise;
    int64_t noise_stride;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* out_symbols;
    float* out_logprobs;
    void* workspace;
    uint64_t workspace_bytes;
} LeoSample;
int32_t leo_sample_workspace_bytes(uint64_t rows, uint64_t symbols, uint64_t* bytes);
int32_t leo_sample(const LeoSample* sample, void* stream);

#ifdef __cplusplus
}
#endif

#endif
