/*
 * leo_decode.h -- C-ABI of the operators that take a model from activations to
 * its next symbol: matrix-vector products with 4-bit weights and group scales
 * (the readout of a served model), the control of logits (penalties for
 * repeated symbols, biases, grammar masks) and the draw of one symbol a row; and
 * of those that answer with several hypotheses at once: products with 8-bit
 * weights and activations, the selection of beams and the reordering of their states.
 *
 * Same manner as leo_hip.h: every call returns an int32 status (0 = ok) and
 * leo_hip_last_error() returns the message of the last failure on the calling
 * thread. All pointers inside the argument structs (but LeoReorder's `arrays`) are
 * device memory of the device that `stream` (a hipStream_t; NULL = the default stream) belongs to,
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
 * x share no memory, nor do y and the bias but where y is one row of floats and the
 * bias itself. `workspace`: at least leo_q4_workspace_bytes()
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

/* An 8-bit weight matrix [outputs, inputs]: w[n, k] = scale[n] * code[n, k] with
 * codes -128..127 and at most 2^27 inputs. */
typedef struct LeoQ8Shape {
    uint64_t outputs;
    uint64_t inputs;
} LeoQ8Shape;

/* Bytes of the device layout that leo_q8_layout writes. */
int32_t leo_q8_layout_bytes(const LeoQ8Shape* shape, uint64_t* bytes);

/* Lays a matrix out once for leo_q8_matmul. codes: int8, codes_stride from row to
 * row; scales: `outputs` values of scale_type. `layout` (256-byte aligned)
 * receives layout_bytes. */
typedef struct LeoQ8Source {
    LeoQ8Shape shape;
    const void* codes;
    int64_t codes_stride;
    const void* scales;
    int32_t scale_type; /* LEO_TYPE_* */
    uint32_t pad0;
    void* layout;
    uint64_t layout_bytes;
} LeoQ8Source;
int32_t leo_q8_layout(const LeoQ8Source* source, void* stream);

/* y[m, n] = bias[n] + s[m] * scale[n] * sum over k of q[m, k] * code[n, k], where
 * s[m] is the larger of 2^-126 and the largest magnitude of row m of x times the
 * float nearest to 1 / 127, rounded to float, and q[m, k] the whole number nearest to
 * x[m, k] / s[m], of two the even one. Sums of codes are exact; rounded to float they
 * are multiplied by scale[n], which has to leave a finite float, then by s[m] with the
 * bias in one fused operation, and rounded to y_type. A row of x with an infinity or
 * NaN gives NaN. bias (float) may be NULL. y and x share no memory, nor do y and the bias
 * but where y is one row of floats and the bias itself. Results whose launch
 * would have 2^32 threads, 2^28 outputs or more, may be refused. `workspace`: at least
 * leo_q8_workspace_bytes() bytes (none where that is 0), 256-byte aligned, whatever
 * they hold; free again when the call's work is done. */
typedef struct LeoQ8Product {
    LeoQ8Shape shape;
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
} LeoQ8Product;
int32_t leo_q8_workspace_bytes(const LeoQ8Shape* shape, uint64_t rows, int32_t x_type, uint64_t* bytes);
int32_t leo_q8_matmul(const LeoQ8Product* product, void* stream);

/* Beam search's selection, `groups` searches of `beams` hypotheses each (65,535
 * hypotheses at most). logits has a row of `symbols` (2^26 at most) for each
 * hypothesis, scores [groups, beams] the sums of log probabilities so far, -inf where
 * there is none (NaN counts as -inf). Candidates:
 *     symbol v after hypothesis b:  score + z[v] - log sum exp z  (those above -inf)
 *     a finished hypothesis itself:  its score; its logits do not count
 * and the `kept` (at most 64, as are the beams) with the largest score / length^length_penalty
 * are taken, largest first; of equals the lower hypothesis, the larger logit, the
 * lower symbol. length counts the symbol that comes in: lengths[b] + 1, lengths[b]
 * of a finished one, at least 1; lengths may be NULL where length_penalty is 0.
 * Logits count as in leo_sample, those of +inf share all probability. Ranks are
 * held in 64 bits; the log of a row's sum is off by up to 2^-21, the same for all of its
 * symbols.
 * out_parents is the hypothesis within its search; out_symbols is -1 for a finished
 * one. Places that no candidate takes have symbol -1, parent 0 and score -inf.
 * finished (bytes, 0 or not) may be NULL: none is. out_finished (may be NULL) is 1
 * for finished ones and where the symbol is `end` (-1: no symbol ends), else 0;
 * out_lengths (may be NULL, needs lengths) the lengths, hypothesis 0's at places that
 * no candidate takes. Outputs have [groups, kept] entries and share no memory with
 * inputs or each other. `workspace` as in leo_q4_matvec. */
typedef struct LeoBeams {
    uint64_t groups;
    uint64_t beams;
    uint64_t kept;
    uint64_t symbols;
    const void* logits;
    int64_t logits_stride;
    int32_t type;
    uint32_t pad0;
    const float* scores;
    const uint8_t* finished;
    const int32_t* lengths;
    double length_penalty;
    int64_t end;
    int32_t* out_symbols;
    int32_t* out_parents;
    float* out_scores;
    uint8_t* out_finished;
    int32_t* out_lengths;
    void* workspace;
    uint64_t workspace_bytes;
} LeoBeams;
int32_t leo_beam_workspace_bytes(uint64_t groups, uint64_t beams, uint64_t kept, uint64_t symbols, uint64_t* bytes);
int32_t leo_beam_select(const LeoBeams* beams, void* stream);

/* Rows of `count` arrays in the order of their parents: row g * kept + k of the target
 * becomes row g * beams + parents[g, k] of the source, zeros where the parent is
 * outside 0 .. beams-1. A row is `outer` pieces of `width` bytes; strides are
 * bytes, not negative. An array may be its own target (same address and strides,
 * kept = beams); otherwise no target shares memory with the parents, any source or
 * other target, which arrays that interleave have to show by common divisors of their
 * strides.
 * `arrays` is host memory, read during the call. */
typedef struct LeoStateArray {
    const void* source;
    void* target;
    uint64_t outer;
    uint64_t width;
    int64_t source_row;
    int64_t source_outer;
    int64_t target_row;
    int64_t target_outer;
} LeoStateArray;
typedef struct LeoReorder {
    const LeoStateArray* arrays;
    uint64_t count;
    uint64_t groups;
    uint64_t beams; /* at most 64, as is kept */
    uint64_t kept;
    const int32_t* parents; /* [groups, kept] */
} LeoReorder;
int32_t leo_reorder_states(const LeoReorder* reorder, void* stream);

#ifdef __cplusplus
}
#endif

#endif
