/*
 * iq.h -- C ABI of the MI355X (gfx950) quantized-weight matrix path.
 *
 * Drop-in boundary for the quantised part of the reference's device ABI
 * (RyanXiaoo/infer kernels/ops/ops.cuh:165-178).  Plain C: no HIP, CUDA or
 * torch types; device memory is passed as plain pointers owned by the caller,
 * the stream as an opaque pointer (a hipStream_t; NULL = the null stream).
 *
 * Layout (the reference's src/quant.h:34-58, produced by src/quant.cpp and
 * tools/quantize.cpp), one [rows x cols] matrix, row-major, groups of
 * IQ_GROUP consecutive columns along a row:
 *   q       int8: rows*cols bytes (two's complement codes -127..127)
 *           int4: rows*cols/2 bytes, element (r,c) in byte (r*cols+c)/2,
 *                 low nibble when c is even (codes 0..15)
 *   scales  bf16 bits, rows x ceil(cols/128)
 *   zeros   int4 only: u8 zero points, rows x ceil(cols/128); NULL for int8
 *   dequant: int8 w = s*q ; int4 w = s*(q - z)          (src/quant.cpp:86-93)
 *
 * Every entry point enqueues work on `stream` and returns without
 * synchronising.  Return value: 0 on success, a negative IQ_E* code when the
 * arguments are rejected on the host (nothing was enqueued), or a positive
 * hipError_t when the HIP runtime reported an error.  No exception crosses
 * this boundary.  The library keeps one workspace (activation operands,
 * split-K partial sums, the prefill GEMM's prepared operands; about 167 MB)
 * per (device, stream) pair, allocated by iq_init / iq_init_stream or on the
 * first call on that stream: calls on different streams may overlap, and
 * calls on one stream are ordered by the stream.  After that no call
 * allocates, frees or synchronises, so any call can be graph-captured the
 * first time it is made.  A stream under graph capture cannot allocate: a
 * call on a capturing stream that has no workspace yet (no iq_init_stream
 * before the capture) returns an error and enqueues nothing.  A captured
 * graph uses the workspace of the stream it was captured on: its replays have
 * to be ordered with that stream's calls and with other graphs captured on it.
 */
#ifndef IQ_H
#define IQ_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IQ_GROUP 128

/* gpu::QuantKind (kernels/ops/ops.cuh:165): kInt8 = 0, kInt4 = 1. */
enum { IQ_INT8 = 0, IQ_INT4 = 1 };

/* Error codes (negative). */
enum {
    IQ_OK = 0,
    IQ_EKIND = -1,      /* kind is neither IQ_INT8 nor IQ_INT4 (a cache's type: IQ_KV_*) */
    IQ_ESHAPE = -2,     /* inconsistent or unsupported sizes */
    IQ_ENULL = -3,      /* a required pointer is NULL */
    IQ_ETOOLARGE = -4,  /* problem exceeds the workspace limits */
    IQ_ENOMEM = -5,     /* workspace allocation failed */
    IQ_EDEVICE = -6,    /* no usable gfx950 device, or not the chain's device */
    IQ_EALIAS = -7      /* an output overlaps an input */
};

/* gpu::QuantView (kernels/ops/ops.cuh:166-172), byte-compatible on LP64:
 * a 4-byte kind, 4 bytes padding, then rows/cols/groups and three pointers. */
typedef struct iq_view {
    int32_t kind;
    int64_t rows, cols, groups;  /* groups = ceil(cols / 128) */
    const uint8_t* q;
    const uint16_t* scales;
    const uint8_t* zeros;        /* int4: rows*groups bytes; int8: NULL */
} iq_view;

/* y[b, o] = sum_c dequant(W, o, c) * x[b, c] (+ bf16 bias[o]), b < B, o < out.
 * Replaces launch_gemv_batched_q (kernels/ops/ops.cuh:173-174,
 * kernels/ops/quant.cu:312-345).  1 <= B <= 32.  x is fp32 [B][in]
 * (only B rows are read; the reference reads up to 32), y fp32 [B][out]
 * (only B rows are written).  in == W->cols, out == W->rows.  bias may be NULL. */
int iq_gemv(const float* x, const iq_view* W, const uint16_t* bias, int B, int64_t in,
            int64_t out, float* y, void* stream);

/* iq_gemv without any allocation, for callers that cannot allocate device
 * memory (code under HIP graph capture, serving loops and harnesses that
 * forbid hipMalloc).  No counterpart in the reference.  Same contract and
 * kernels as iq_gemv, limited to in <= 32768 (IQ_ETOOLARGE beyond), with
 * its scratch (activation operands and split-K partial sums, ~20.1 MiB) in
 * a static device array of the library that each device holds until the
 * process ends.  Every call on a device shares that array, whatever the
 * stream: calls that overlap in time on one device race, so order them
 * (e.g. one stream).  No state carries from one call to the next. */
int iq_gemv_noalloc(const float* x, const iq_view* W, const uint16_t* bias, int B, int64_t in,
                    int64_t out, float* y, void* stream);

/* The two halves of iq_gemv, for callers that multiply one activation
 * block by several matrices (q/k/v, gate/up share their input):
 * iq_gemv_prep takes x [B][in] (fp32) once into the device workspace: a
 * copy for B <= 4 (the GEMV kernel converts it itself), otherwise per row
 * and 128-column group a power-of-two scale 2^-k and x * 2^k as two fp16
 * terms (or as four signed byte limbs of rint(x * 2^k)), in the column
 * order that `kind`'s weight unpacking produces;
 * iq_gemv_prepped then runs the GEMV of any matrix of that kind and width on
 * the prepared block.  A prepared block belongs to the stream it was made
 * on and stays valid until the next iq_gemv_prep on that stream, or until
 * an iq_gemv / iq_gemv_multi / iq_linear on that stream reuses its buffers.
 * iq_gemv_prepped returns IQ_ESHAPE when there is no valid preparation or
 * (B, in, kind) differ from it.
 * No reference counterpart: the reference's launcher re-reads x per matrix. */
int iq_gemv_prep(const float* x, int B, int64_t in, int kind, void* stream);
int iq_gemv_prepped(const iq_view* W, const uint16_t* bias, int B, int64_t in, int64_t out,
                    float* y, void* stream);

/* iq_gemv_prepped for n <= 4 matrices of one kind and width at once
 * (y_i = x * W_i^T + bias_i, out_i = Ws[i]->rows): q|k|v or gate|up of a
 * layer in one launch.  The reference runs them as separate launches
 * (kernels/batch_gpu.cu:192-194,210-211) and fuses only bf16 weights
 * (kernels/model_gpu.cu:31-38).  biases may be NULL (no bias anywhere) or
 * hold NULL entries. */
int iq_gemv_prepped_multi(const iq_view* const* Ws, int n, const uint16_t* const* biases, int B,
                          int64_t in, float* const* ys, void* stream);

/* iq_gemv for n <= 4 matrices of one kind and width sharing the activations
 * x [B][in]: one GEMV launch reads x and all n matrices (at B <= 4 the
 * activation conversion happens inside it; at larger B a conversion launch
 * precedes it, and split-K shapes add a reduction launch).  Same matrix/bias
 * conventions as iq_gemv_prepped_multi; the prepared block of the workspace
 * may be overwritten.  No reference counterpart (see iq_gemv_prepped_multi). */
int iq_gemv_multi(const float* x, const iq_view* const* Ws, int n, const uint16_t* const* biases, int B,
                  int64_t in, float* const* ys, void* stream);

/* Same contract for any T >= 1 (fp32 activations).  Replaces
 * launch_gemm_tiled_q (kernels/ops/ops.cuh:175-176, kernels/ops/quant.cu:347-351).
 * Runs the MFMA prefill GEMM with the activations split into bf16 hi + lo. */
int iq_gemm(const float* x, const iq_view* W, const uint16_t* bias, int64_t T, int64_t in,
            int64_t out, float* y, void* stream);

/* Prefill GEMM with bf16 activations x [T][in] (bf16 bits), fp32 output.
 * No reference counterpart (the reference's activations are fp32); it is the
 * bf16-activation form of iq_gemm used for the Qwen2.5-7B prefill shapes. */
int iq_gemm_bf16x(const uint16_t* x, const iq_view* W, const uint16_t* bias, int64_t T,
                  int64_t in, int64_t out, float* y, void* stream);

/* The quantised linear call site, GpuBatch::Impl::linear_b
 * (kernels/batch_gpu.cu:137-147): T <= 32 -> iq_gemv, T > 32 -> iq_gemm. */
int iq_linear(const float* x, const iq_view* W, const uint16_t* bias, int64_t T, int64_t in,
              int64_t out, float* y, void* stream);

/* out[t, i] = dequant(table, ids[t], i), exactly.  Replaces launch_embedding_q
 * (kernels/ops/ops.cuh:177-178, kernels/ops/quant.cu:304-309,353-357).
 * H == table->cols.  An id outside [0, rows) yields a row of NaN (the
 * reference reads out of bounds). */
int iq_embedding(const iq_view* table, const int64_t* ids, int64_t T, int64_t H, float* out,
                 void* stream);

/* On-device quantize + pack of a bf16 [rows x cols] matrix, bit-exact to
 * llm::quantize (src/quant.cpp:34-84, src/quant.h:61), which the reference
 * runs on the CPU only (tools/quantize.cpp:30-49).  Writes q, scales and (int4)
 * zeros in the layout above.  int4 needs even cols (as the reference). */
int iq_quantize(const uint16_t* w_bf16, int64_t rows, int64_t cols, int kind, uint8_t* q,
                uint16_t* scales, uint8_t* zeros, void* stream);

/* ---------------------------------------------------------------- chains
 * A chain is a program of dependent GEMV stages of 1..32 activation rows:
 * the quantised linears of a (batched) decode step in the order of
 * GpuBatch::Impl::launch_sequence (kernels/batch_gpu.cu:186-215), each
 * stage reading what earlier stages wrote, with the elementwise work
 * between them fused into the stages.  A run is one launch per 1-row stage
 * and one or two per B-row stage (the GEMV with the input transform, and on
 * long rows the K-range sums with the output transform), on one stream, capturable into
 * a HIP graph.  No reference counterpart as an entry point: the reference
 * issues launch_gemv_batched_q, launch_rmsnorm, launch_swiglu and
 * launch_residual_add separately.
 *
 * Stage = y_i = f_out( dequant(W_i) . f_in(x) + bias_i ), i < n <= 3, all W_i
 * of one kind and width K (K % 256 == 0; 1 row: int4 K <= 24576, int8
 * K <= 20480, halved for IQ_OUT_SWIGLU), x 16-byte aligned, for each of
 * the stage's `rows` activation rows B (1..32; 0 means 1): x is [B][K]
 * ([B][K / group] for IQ_IN_GQA), residual and every y_i [B][W_i->rows],
 * row-major, each row transformed on its own (RMSNorm per row):
 *   f_in   IQ_IN_PLAIN    x[k]
 *          IQ_IN_RMSNORM  x[k] / sqrt(mean(x^2) + eps) * norm[k], norm bf16
 *                         (src/forward.cpp:21-31); K <= 16384
 *          IQ_IN_GQA      x[(k / (head_dim * group)) * head_dim + k % head_dim]:
 *                         the attention output of a sequence of one token,
 *                         whose softmax over its single key is 1, so every
 *                         query head receives the value row of its key/value
 *                         head (x = v, K / group values)
 *   f_out  IQ_OUT_STORE     y_i[o] = acc + bias_i[o]
 *          IQ_OUT_RESIDUAL  y_0[o] = residual[o] + (acc + bias_0[o])  (n == 1)
 *          IQ_OUT_SWIGLU    y_0[o] = silu(acc_0 + b_0) * (acc_1 + b_1), n == 2
 *                           (gate, up; kernels/ops/elementwise.cu:6-11)
 * A stage's outputs may not overlap its own inputs (IQ_EALIAS).  Outputs
 * are fp32 vectors of W_i->rows. */
enum { IQ_IN_PLAIN = 0, IQ_IN_RMSNORM = 1, IQ_IN_GQA = 2 };
enum { IQ_OUT_STORE = 0, IQ_OUT_RESIDUAL = 1, IQ_OUT_SWIGLU = 2 };

typedef struct iq_stage {
    int32_t in_op, out_op, n;
    int32_t gqa_head_dim, gqa_group;  /* IQ_IN_GQA */
    float eps;                        /* IQ_IN_RMSNORM */
    const float* x;
    const uint16_t* norm;             /* IQ_IN_RMSNORM: bf16 [K], 16-byte aligned */
    const float* residual;            /* IQ_OUT_RESIDUAL: [rows] */
    iq_view W[3];
    const uint16_t* bias[3];          /* bf16 or NULL */
    float* y[3];                      /* IQ_OUT_SWIGLU: y[0] only */
    int32_t rows;                     /* activation rows B, 1..32 (0: 1) */
} iq_stage;

typedef struct iq_chain iq_chain;

/* Validates the n stages and records their launch shapes for the current
 * device.  The chain allocates its own device buffers here: the sums of
 * squares passed from a stage to a later RMSNorm stage (a float per 16-row
 * tile, or per row and tile / 256-column block with rows > 1), and for
 * stages with rows > 1 the K-range partial sums of the rows GEMV and the
 * prepared f16 operands of narrow stages (5..16 rows: G * 8 KiB).  So
 * create a chain outside graph capture, in code that may allocate;
 * iq_chain_destroy frees them.  iq_chain_run allocates nothing. */
int iq_chain_create(const iq_stage* stages, int n, iq_chain** out);
/* Enqueues one run of the whole program on `stream`. */
int iq_chain_run(const iq_chain* chain, void* stream);
void iq_chain_destroy(iq_chain* chain);

/* ------------------------------------------------ the cache of a decode step
 * A paged key/value cache, the attention of one new token a sequence over
 * it, and eviction from it.  No counterparts in the reference's quantised
 * path; iq_attn_decode's output is what a chain stage with IQ_IN_PLAIN reads
 * (the o projection), its q and the appended k, v are what the q|k|v stage
 * writes.
 *
 * A sequence's token t (0 <= t < its length) lies in slot t % page_size of
 * page table[b][t / page_size]; its key vector for key/value head h starts at
 *   k + page * page_stride + slot * slot_stride + h * head_stride
 * (in elements; v alike), head_dim contiguous values.  Any order of pages,
 * slots and heads in memory can be described, and pages may be shared between
 * sequences as long as nothing writes them.  k, v 16-byte aligned, the strides
 * multiples of 8, head_dim a multiple of 8 in 8..256 (8-bit types: of 16).
 *
 * A cache holds bf16 or fp16 values, or 8-bit codes (signed integers
 * -127..127, or e4m3 numbers up to 448) with a scale for every `block`
 * consecutive slots of a page and key/value head: the value of a code is code *
 * scale.  iq_kv_append, iq_attn_decode and iq_kv_evict take 16-bit caches
 * (IQ_EKIND); iq_kv_extend, iq_kv_read and iq_attn_decode_window take all.
 * What a call makes for its caller (q_out, out, k_out, v_out) must not overlap
 * the cache's rows or scales (IQ_EALIAS); between them, in a larger tensor, it
 * may lie. */
enum { IQ_KV_BF16 = 0, IQ_KV_F16 = 1, IQ_KV_I8 = 2, IQ_KV_E4M3 = 3 };

typedef struct iq_kv {
    int32_t type;                              /* IQ_KV_* */
    int32_t kv_heads, head_dim, page_size;     /* page_size: any number of slots >= 1 */
    int64_t pages;                             /* in the pool, < 2^31 */
    int64_t page_stride, slot_stride, head_stride;
    void* k;
    void* v;
} iq_kv;

/* The scales of an 8-bit cache: that of slot s of a page and head h is at
 *   k + page * page_stride + (s / block) * block_stride + h * head_stride
 * (in floats; v alike).  block divides page_size (1: a scale for each token
 * and head). */
typedef struct iq_kv_scales {
    int32_t block;
    int64_t page_stride, block_stride, head_stride;
    float* k;
    float* v;
} iq_kv_scales;

/* Adds T >= 1 tokens to the cache: k, v fp32 [T][kv_heads][head_dim] are written
 * to slot slots[t] = page * page_size + slot (rounded to the cache's type,
 * to nearest even), q fp32 [T][q_heads][head_dim] goes to q_out; q and k with
 * rotary embedding on their first rot_dim values (pairs i, i + rot_dim/2
 * turned by positions[t] * freqs[i], freqs double [rot_dim/2]; angles in
 * 64 bits, so far positions keep their precision).  rot_dim: a multiple of 8
 * up to head_dim, or 0 (no rotation; positions and freqs unused).  A slot
 * outside the pool (e.g. -1, a padded row) writes nothing to the cache; two
 * tokens of one call must not have the same slot.  q_out may be q itself;
 * another overlap of q_out with q, k or v is refused (IQ_EALIAS).  q and q_out
 * may be NULL with q_heads = 0. */
int iq_kv_append(const float* q, const float* k, const float* v, const int64_t* positions, const int64_t* slots,
                 int64_t T, int q_heads, const double* freqs, int rot_dim, const iq_kv* kv, float* q_out,
                 void* stream);

/* Attention of one token a sequence over its cached tokens:
 *   p[b,h,t] = softmax over t < lens[b] of scale * q[b,h] . key[b,t,h / g]
 *   out[b,h] = sum_t p[b,h,t] value[b,t,h / g],   g = q_heads / kv_heads
 * q, out fp32 [B][q_heads][head_dim] (out must not overlap q), table int32
 * [B][table_ld] of which the first max_pages entries of a row may be used
 * (entries past a sequence's last page are not read), lens int32 [B], 1 <= B
 * <= 1024.  Scores, softmax and sums are fp32; the 16-bit keys and values
 * are taken as they are (over an fp16 cache, q and p enter the products to
 * 2^-23 of themselves, and to 2^-38 of the head's largest |q| and 2^-37 of its
 * largest p).  Keys and values past a sequence's length have no influence,
 * whatever they hold.
 * weights (may be NULL): fp32 [B][kv_heads][weights_ld], weights_ld >=
 * max_pages * page_size; weights[b][j][t] += sum over the heads h of key/value
 * head j of p[b,h,t], for t < lens[b]; the rest is left as it was.  The
 * scores lie in the workspace, as much room a sequence as its table row can
 * hold tokens: max_pages * page_size * q_heads may be at most 20971520 with
 * weights (IQ_ETOOLARGE), and of a larger batch 20971520 / (max_pages *
 * page_size * q_heads) sequences go at a time, one group behind the other
 * however short they are.  Where weights are wanted, max_pages should be no
 * more than the longest sequence needs.
 * A sequence of length 0 gives zeros.  A length below 0 or above max_pages *
 * page_size gives NaN, its weights left as they were.  A page id outside [0,
 * pages) among the sequence's pages, a q that is not finite or a key of NaN
 * gives NaN to the heads that read it and to the weights made of them; a value
 * that is not finite gives NaN (or its infinity) to the heads.  Scores are fp32
 * numbers, in powers of 2: one below fp32's range (-inf) weighs nothing, and a
 * head with no other scores gives zeros and adds nothing to the weights; one
 * above it (+inf), or made of products past the range with both signs, is like
 * NaN.  An infinite key gives one or the other. */
int iq_attn_decode(const float* q, const iq_kv* kv, const int32_t* table, int64_t table_ld, int64_t max_pages,
                   const int32_t* lens, int B, int q_heads, float scale, float* out, float* weights,
                   int64_t weights_ld, void* stream);

/* Cuts every sequence of more than `budget` tokens to `budget`, for each
 * key/value head by itself: of its n = lens[b] tokens stay the newest `recent`
 * (0 <= recent <= budget) and, of the n - recent older ones, the budget -
 * recent of the largest weights[b][h][t] (equal ones: the lower t; NaN counts
 * as less than any number).  With cut = budget - recent: a kept older token
 * below cut stays where it is, the kept ones above it fill the free places
 * below cut, both in ascending order, and the newest follow in their order.
 * "Newest" goes by place: the last `recent` slots.  Tokens appended one after
 * the other lie in the order of their age; behind a call that cut the sequence
 * only its last `recent` ones and those appended since do, so `recent` must not
 * be more than these at the next call (a larger one keeps the tokens in the last
 * slots, which are then not the newest; the device holds the lengths, so this
 * is not checked).  weights move along, and weights[b][h][t] = 0 for budget <= t < n, so that a
 * slot appended later starts at 0.  new_lens[b] = min(lens[b], budget) for
 * every head alike (the pages past it are free); it must not overlap lens.
 * Pages must not be shared between the sequences of a call nor appear twice in
 * one.  The lists of what moves lie in the workspace: min(budget - recent,
 * max_pages * page_size - budget) * kv_heads may be at most 8 million
 * (IQ_ETOOLARGE).  A sequence whose
 * length is below 0 or above max_pages * page_size, or any of whose first
 * ceil(n / page_size) page ids lies outside [0, pages), is left as it is and
 * its new length is its old one.  1 <= B <= 1024, budget >= 1; table, lens and
 * weights as above. */
int iq_kv_evict(const iq_kv* kv, const int32_t* table, int64_t table_ld, int64_t max_pages, const int32_t* lens,
                int B, int64_t budget, int64_t recent, float* weights, int64_t weights_ld, int32_t* new_lens,
                void* stream);

/* Adds T new tokens of B sequences behind what each has cached, the first
 * lens[b] tokens in the pages table[b]: rows starts[b] <= t < starts[b + 1] of q,
 * k, v and positions are sequence b's tokens lens[b], lens[b] + 1, ... (starts
 * int32 [B + 1], ascending, from 0 to T; NULL: one token each, T = B).  lens is read
 * only: the sequence's length is lens[b] + its new tokens afterwards.
 *   norms     q_norm, k_norm (bf16 [head_dim], each may be NULL): every head of q
 *             (k) becomes x / sqrt(mean(x^2) + eps) * norm first, eps >= 0
 *   rotation  as in iq_kv_append, behind the norms
 *   q         goes to q_out in fp32 (every row below T, whatever its sequence)
 *   k, v      are rounded into the cache, to nearest even
 * A token behind the table's last page, in a page whose id lies outside [0,
 * pages) or of a sequence whose length is below 0 or above max_pages * page_size is
 * not stored.  Rows that belong to no sequence are not either.  The pages that a
 * call writes must be different ones (a row of the table may name a page again
 * once no token of its earlier place is read any more, as under a window).
 *
 * An 8-bit cache's blocks start anew with their first slot: with a = max |x| over
 * the call's tokens of the block (one head's k or v), in fp32, and Q = 127 (448),
 *   - a block whose first slot is among them, or whose scale is not above 0, gets the
 *     scale s = max(a / Q, 2^-126), or 0 if a is 0;
 *   - a block that holds older tokens (the sequence's, below lens[b]) keeps its
 *     scale if a <= Q * s; otherwise s doubles until it is so and the older
 *     tokens' codes are halved as often, at once, to nearest even.  So a stored
 *     value is off by less than one step of its block's scale (int8; half a
 *     step where the scale did not grow), however often it grew.  The comparison
 *     is exact and s a quotient rounded to nearest: where Q * s came out below the
 *     a that made it (two in five to one half of all a), the same a in a later call
 *     doubles the scale, once.  Tokens of one call, and blocks of one slot, do not
 *     meet this.
 * A unit of work is a block's tokens of a call and one key/value head: blocks of
 * 8 to 64 slots are fast, larger ones leave few units of many steps, and a scale that
 * grows costs its block's older tokens read and written.
 * Codes are x / s to nearest even.  A value that is not finite makes its block's
 * scale NaN, and all that is read from the block, until the block starts anew. */
int iq_kv_extend(const float* q, const float* k, const float* v, int64_t T, int q_heads, const uint16_t* q_norm,
                 const uint16_t* k_norm, float eps, const int64_t* positions, const double* freqs, int rot_dim,
                 const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table, int64_t table_ld,
                 int64_t max_pages, const int32_t* lens, const int32_t* starts, int B, float* q_out, void* stream);

/* Cached tokens back as numbers: rows starts[b] <= t < starts[b + 1] of k_out
 * and v_out ([T][kv_heads][head_dim], 16-byte aligned, one of them may be NULL) become sequence
 * b's tokens first[b], first[b] + 1, ... (first NULL: 0).  out_type IQ_READ_*; a
 * code times its scale is an fp32 product, then rounded to the type, both to
 * nearest even.  Rows that belong to no
 * sequence are left as they were; a token outside the table, or in a page whose
 * id lies outside [0, pages), is NaN. */
enum { IQ_READ_F32 = 0, IQ_READ_BF16 = 1, IQ_READ_F16 = 2 };
int iq_kv_read(const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table, int64_t table_ld, int64_t max_pages,
               const int32_t* first, const int32_t* starts, int B, int64_t T, int out_type, void* k_out, void* v_out,
               void* stream);

/* iq_attn_decode, without weights, over a cache of any type (scales: of an
 * 8-bit one; not used otherwise), and optionally under a window: with window > 0 a
 * sequence sees its newest `window` tokens and its first `sinks` ones, t >= lens[b]
 * - window or t < sinks.  Pages that hold none of these are not read, and their
 * table entries may be anything.  window = 0: all tokens, whatever sinks is.
 * Keys and values are the codes times their scales, in fp32: a scale of a key
 * multiplies its score, that of a value its weight (in full precision from scales of
 * 2^-86 on).  A NaN or infinite scale is like a NaN key or value. */
int iq_attn_decode_window(const float* q, const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table,
                          int64_t table_ld, int64_t max_pages, const int32_t* lens, int B, int q_heads, float scale,
                          int64_t window, int64_t sinks, float* out, void* stream);

/* Log probabilities over rows of logits, fp32 [T][V] with `ld` >= V floats
 * from row to row (V < 2^31 - 65536):
 *   logprob[t]  log softmax(row t)[tokens[t]]; NaN for a token outside [0, V)
 *   entropy[t]  -sum p log p
 *   top_ids[t][i], top_logprobs[t][i], i < top <= 64: the `top` largest, by
 *               value descending, equal ones by id ascending
 * tokens and logprob are NULL together, entropy may be NULL, top_ids and
 * top_logprobs are NULL with top = 0; at least one output is asked for and
 * top <= V.  A logit of -inf has probability 0 and log probability -inf.  A
 * row that holds NaN or +inf, or nothing but -inf, has no distribution: its
 * log probabilities and entropy are NaN (its ids are still ranked, NaN as the
 * largest). */
int iq_logprobs(const float* logits, int64_t ld, int64_t T, int64_t V, const int64_t* tokens, int top,
                float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, void* stream);

/* Reserve the workspace of (device, null stream) (done lazily by the first
 * call that needs it).  Call before capturing a graph.  Returns 0 or an
 * error code. */
int iq_init(int device);

/* Reserve the workspace of (device, stream): call before capturing a graph
 * on a stream other than the null stream, since capture forbids the
 * allocation.  Library set-up, no reference counterpart (the reference's
 * launchers keep no workspace). */
int iq_init_stream(int device, void* stream);

/* Static description of an error code (never NULL). */
const char* iq_error_string(int code);

/* Library version string. */
const char* iq_version(void);

#ifdef __cplusplus
}
#endif

#endif /* IQ_H */
