/* The device primitive ABI of cmachine's Qwen runtime, implemented for B200.
 *
 * This header replaces the reference's src/gpu.h: a C caller written against
 * that header (the reference's src/qwen.c, src/bounded_cache.h, tests) links
 * against libcmachine_b200.so unchanged. Every prototype keeps the reference's
 * name, argument order and meaning; the line after each group cites the
 * reference declaration it replaces. Semantics kept from the reference:
 *   - all pointers are device pointers owned by the caller; gpu_alloc'd blocks
 *     are tracked process-wide and gpu_free of an unknown pointer is fatal
 *     (src/qwen_cuda.cu:13-19);
 *   - any CUDA error is fatal: message on stderr, exit(2) (src/qwen_cuda.cu:8);
 *   - gpu_top2 exits(2) on non-finite input (src/qwen_cuda.cu:117);
 *   - work is ordered as one stream: gpu_read returns data written by every
 *     earlier call.
 * What differs: no cuBLAS (hand-written sm_100a kernels), BF16 matrices are
 * read directly (no FP32 tile), and matvec/attention use FP32 with fused
 * multiply-add in a fixed parallel order, so results match the reference to
 * tolerance rather than bit for bit. Every kernel is deterministic: the same
 * inputs give the same bits on every call.
 */
#ifndef TCM_GPU_H
#define TCM_GPU_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

typedef struct TcmGpu TcmGpu;
/* Top-2 of a vector: ids and values; ties go to the lower id. (src/gpu.h:9) */
typedef struct { int first, second; float first_value, second_value; } TcmTop2;

/* Handle with per-caller scratch (top-2 partials, flags). (src/gpu.h:10-11) */
TcmGpu *gpu_open(void);
void gpu_close(TcmGpu *);

/* Tracked device memory and copies. (src/gpu.h:12-17, 38, 49-51) */
void *gpu_alloc(size_t bytes);
void gpu_free(void *);
void gpu_zero(void *, size_t bytes);
void gpu_copy(void *dst, const void *src, size_t bytes);   /* device -> device */
void gpu_read(void *host, const void *dev, size_t bytes);  /* device -> host, synchronous */
void gpu_write(void *dev, const void *host, size_t bytes); /* host -> device, synchronous */
void gpu_sync(void);
size_t gpu_live_bytes(void);
size_t gpu_peak_bytes(void);
size_t gpu_free_bytes(void);

/* Upload n host values of dtype 1 (FP32) or 2 (BF16, widened) as FP32. (src/gpu.h:18) */
float *gpu_weight(const void *host, uint32_t dtype, size_t n);

/* y[out] = W[out][in] x, W row-major. If W was registered by gpu_owned_weight
 * under profile 2 it holds BF16 and is read as such. (src/gpu.h:19) */
void gpu_matvec(TcmGpu *, const float *w, int in, int out, const float *x, float *y);
/* out = (x * r) * w, r = rsqrt(mean(x^2) + eps); _scale also stores r. (src/gpu.h:20-23) */
void gpu_rms(float *out, const float *x, const float *w, int n, float eps);
void gpu_rms_scale(float *out, const float *x, const float *w, int n, float eps, float *scale);
/* Experimental elementwise ops of the receiver-plane studies. (src/gpu.h:24-28) */
void gpu_multiply(float *out, const float *x, const float *y, int n);
void gpu_plane(float *out, const float *base, const float *a, const float *b, int n, float s, float t);
void gpu_plane_scaled(float *out, const float *base, const float *a, const float *b, int n, float s, float t,
                      const float *scale);
void gpu_linear2(float *out, const float *a, const float *b, int n, float ca, float cb, const float *scale);
/* 1 when a and b are bitwise equal and finite, else 0. (src/gpu.h:29) */
int gpu_identical_finite(TcmGpu *, const float *a, const float *b, int n);
/* x += y. (src/gpu.h:30-31) */
void gpu_add(float *x, const float *y, int n);
void gpu_bias(float *x, const float *y, int n);
/* Half-split RoPE of `heads` rows of `dim` at `position`. (src/gpu.h:32) */
void gpu_rope(float *x, int heads, int dim, int position, float theta);
/* Row `position` of each head's [capacity][dim] slab <- x. (src/gpu.h:33) */
void gpu_cache(float *cache, const float *x, int heads, int dim, int capacity, int position);
/* GQA attention of qheads query rows over `length` cached rows; query head h
 * reads K/V head h / (qheads / kvheads); scores is scratch. (src/gpu.h:34) */
void gpu_attention(TcmGpu *, float *out, const float *q, const float *keys, const float *values, float *scores,
                   int qheads, int kvheads, int dim, int capacity, int length);
/* gpu_attention for callers that may not allocate device memory while they run
 * (a host that owns all GPU memory through its own pool, a loop that cannot
 * take cudaFree's device-wide synchronisation). No counterpart in the
 * reference. Same result as gpu_attention for dim 128; no scores are written.
 * Its split-K scratch is a fixed 1.2 MB device array inside the library, held
 * by every GPU that loads it: limits are dim == 128, 1 <= kvheads <= 4, at most
 * 8 query heads per KV head, 1 <= length <= capacity; other sizes return -1
 * with a message on stderr and launch nothing. Returns 0 when launched. CUDA
 * errors are fatal (message, exit(2)) as everywhere in this ABI; only sizes and
 * alignment come back as -1. The first call on each device looks up the
 * array's device address, and under the runtime's lazy module loading that is
 * also when the device first holds the array's 1.2 MB: make that first call at
 * start-up, before handing device memory to a pool and before any stream
 * capture. Calls share the array: calls that overlap on the GPU race. */
int gpu_attention_static(float *out, const float *q, const float *keys, const float *values, int qheads,
                         int kvheads, int dim, int capacity, int length);
/* gate = silu(gate) * up. (src/gpu.h:35) */
void gpu_swiglu(float *gate, const float *up, int n);
/* Experimental polynomial gate law. (src/gpu.h:36-38) */
void gpu_gate_anchor(const float *g, float *p, float *first, float *second, float *s, int n);
void gpu_gate_swiglu(float *g, const float *u, const float *source, const float *p, const float *first,
                     const float *second, const float *s, int n);
/* Top-2 of x[0..n). (src/gpu.h:39) */
TcmTop2 gpu_top2(TcmGpu *, const float *x, int n);

/* Process-wide weight residence profile: 0 native FP32, 1 tiled FP32 (kept as
 * native FP32 here: no tile is needed), 2 source BF16 matrices. Choose before
 * load; release after the model is freed. (src/gpu.h:40-48) */
void gpu_weight_configure(int profile);
float *gpu_owned_weight(TcmGpu *, const void *host, uint32_t dtype, size_t count, int rank, int rows, int columns);
size_t gpu_owned_weight_bytes(const float *, size_t count);
void gpu_owned_embedding(float *out, const float *embedding, int token, int width);
void gpu_weight_release(void);
void gpu_weight_info(size_t *matrix, size_t *vectors, size_t *scratch, int *count, unsigned long long *matvecs,
                     unsigned long long *tiles, unsigned long long *embeddings);

/* Byte-codec K/V cache (src/qwen_cache.inc:13,20,35; declared by the reference
 * in src/bounded_cache.h:7-8). Per (kind, KV head) row: scale = max|x|/127 (1
 * when zero) and code = clamp(round(x/scale), +-127). Returns 0, or -1 when the
 * row holds a non-finite value. Layout per layer: K codes [2][capacity][128],
 * V codes [2][capacity][128], scales [kind*2+head][capacity]. */
int gpu_encode_current(signed char *key, signed char *value, float *scales, const float *k, const float *v,
                       int capacity, int position, int *invalid);
void gpu_byte_attention(TcmGpu *, float *out, const float *q, const signed char *key, const signed char *value,
                        const float *scales, float *scores, float *workspace, int capacity, int length);
void gpu_ring_attention(TcmGpu *, float *out, const float *q, const signed char *key, const signed char *value,
                        const float *scales, float *scores, float *workspace, const int *order,
                        const float *weights, int capacity, int length, int weighted);

/* ---- Paged K/V cache of many sequences (no counterpart in the reference) ----
 * One pool of fixed-size pages holds the K and V rows of every sequence; a table
 * names each sequence's pages, so sequences grow, end and share prefixes without
 * copies. The pool, the table and the extents are device memory of the caller;
 * the descriptors are host structures read during the call.
 *
 * keys and values are [pages][kvheads][page][dim]: BF16 (kind 2, round to nearest
 * even), or the byte codec above (kind 3: int8 codes, with scales [2][pages]
 * [kvheads][page], K's then V's). Limits: dim 64 or 128; 1 <= page <= 65536;
 * keys and values 16-byte aligned; kvheads <= 1024; at most (2^28 - 1) / kvheads
 * new rows a sequence. */
typedef struct {
    int kind, pages, page, kvheads, dim;
    void *keys, *values;
    float *scales; /* kind 3 only */
} TcmPagedCache;
/* A ragged batch: sequence s brings the rows starts[s] .. starts[s + 1] - 1 of the
 * callers' row buffers (which have `rows` rows in all) and has lengths[s] rows in
 * the cache counting them, so new row i stands at place lengths[s] - count + i.
 * table[s * table_stride + p] is the page of places p * page .. p * page + page - 1;
 * entries of places that nothing reads or writes may hold anything. max_new and
 * max_length (at most 2^30) are upper bounds of the new rows and the length of any
 * sequence. */
typedef struct {
    int sequences, rows, max_new, max_length; /* sequences <= 65535 */
    const int *starts;  /* [sequences + 1] */
    const int *lengths; /* [sequences] */
    const int *table;   /* [sequences][table_stride] */
    int table_stride;
} TcmPagedBatch;
/* All three return 0 when launched, or -1 with a message on stderr for sizes,
 * strides or alignment they do not take, and launch nothing; they do not wait for
 * the device, but for a call of attention whose scratch grows. What only the device
 * can see is reported in *status (a device word, 4-byte aligned, that the kernels OR
 * into and never clear; may be NULL): 1 a row was appended that the pool cannot hold,
 * 2 a page id outside the pool for a row that was needed, 4 extents that do not fit
 * rows, max_new, max_length or the table, 8 a wait inside the attention ran out
 * (qwen_b200_wait_limit): its outputs are not to be used. A row without a page is
 * not written, reads as zeros and is visible to no query; a sequence with bad
 * extents is left out, its rows of the outputs untouched. Row buffers are FP32,
 * strides count floats from one row to the next (multiples of 4), buffers are
 * 16-byte aligned; rows of no sequence are neither read nor written.
 *
 * Write the new rows: k and v hold [kvheads][dim] a row, `stride` apart (both). A
 * row of one KV head with a non-finite value, or one whose stored form would be
 * infinite (BF16 from 2^128 - 2^119 on, bytes FP32's largest number), is stored as
 * zeros and reported; bytes hold the ring's codes and scales, but for a row whose
 * max|x| / 127 underflows: the ring refuses it, here it is stored as zeros with
 * scale 0. New rows at negative places (count > length) are skipped. What two
 * sequences of one call that write the same row of a shared page leave there is
 * unspecified. */
int gpu_paged_append(const TcmPagedCache *, const TcmPagedBatch *, const float *k, const float *v, long long stride,
                     int *status);
/* Read the same rows back as the FP32 values they stand for. */
int gpu_paged_read(const TcmPagedCache *, const TcmPagedBatch *, float *k, float *v, long long stride, int *status);
/* Grouped-query attention of the new rows' queries over the cache: the query at
 * place p sees rows j <= p with window == 0, j > p - window or j < sinks, scores
 * q . k / sqrt(dim). q and out hold [qheads][dim] a row; query head h reads KV head
 * h / (qheads / kvheads); at most 8 query heads per KV head. A query that sees no
 * row gets zeros. Outputs that see a row with a non-finite value are unspecified;
 * no other output is touched by it.
 * Precision: FP32 in and out, for magnitudes of queries and rows up to 1e30. The
 * tensor cores get queries and weights as parts of 22 bits or more: over byte rows
 * queries are 23 bits of the row's largest element for few new rows and FP16 pairs
 * for chunks, weights FP16 pairs; over BF16 rows three BF16 parts for few new rows,
 * FP16 pairs for chunks. A weight's step is 2^-28 of the size (max |v|) of the row
 * that counts most for the query, whatever rows within 2^100 of it hold, seen or
 * not. At most 32 truncating steps of 16 rows follow one another; longer sums are
 * FP32, rounded to nearest.
 * Deterministic, but a sequence's result depends on its batch in the last bits.
 * Scratch belongs to the handle and grows on demand, to some 165 MB at most; a call
 * that grows it allocates and waits for the device. Calls with one handle follow one
 * another on the library's stream, and another thread needs a handle of its own. */
int gpu_paged_attention(TcmGpu *, float *out, long long out_stride, const float *q, long long q_stride,
                        const TcmPagedCache *, const TcmPagedBatch *, int qheads, int window, int sinks, int *status);

/* What stands between a projection and the cache: the queries and keys of each head
 * normed (y = x / sqrt(mean x^2 + eps) times qnorm or knorm, [dim] device floats;
 * NULL: not normed) and then rotated to their row's place p: with R = rotary, elements
 * d and d + R / 2, d < R / 2, turn by the angle p theta^(-2d / R); elements from R on
 * stay. rotary is a multiple of 4, at most dim; 0 rotates nothing. */
typedef struct {
    const float *qnorm, *knorm;
    float eps, theta;
    int rotary;
} TcmHeadRotation;
/* gpu_paged_append of rows as a projection leaves them: norms and rotates each new row's
 * queries (into q_out, which may be q with the same stride) and keys, and writes keys
 * and values to the pool as gpu_paged_append does, with its limits, status bits and
 * treatment of rows that the pool cannot hold. q, k and v share one stride; they may be
 * parts of one row. Queries of a row without a page, or at a negative place, are
 * written all the same. Norms, angles and rotations are carried in 64 bits and rounded
 * once to FP32, from which the stored form is taken (gpu_rope's angles are FP32: at
 * place 32768 the two differ by up to 2e-3). A query head with a non-finite value is
 * unspecified, the others are not touched by it. eps is finite and not negative, theta
 * finite and positive; norms are 8-byte aligned. */
int gpu_paged_rotate_append(const TcmPagedCache *, const TcmPagedBatch *, const TcmHeadRotation *, float *q_out,
                            long long q_out_stride, const float *q, const float *k, const float *v, long long stride,
                            int qheads, int *status);
/* Bounds of the keys of each page, for gpu_paged_sparse_attention: bounds is
 * [pages][kvheads][2][dim] BF16 (16-byte aligned), the least and the largest value of
 * every key element over the page's rows, rounded down and up. The call brings every
 * page that holds a new row of the batch up to date, from all rows of the page below its
 * sequence's length; others are not touched. Call it behind each append (a batch whose
 * counts are the lengths does whole sequences). A NaN bounds nothing. What two
 * sequences of one call with different lengths leave of a page that both bring rows of
 * is unspecified. */
int gpu_paged_bounds(const TcmPagedCache *, const TcmPagedBatch *, uint16_t *bounds, int *status);
/* gpu_paged_attention of each query over few pages of its sequence. The query at place p
 * stands in page P = p / page of its sequence. Where P < blocks it sees all rows j <= p.
 * Otherwise every KV head has `blocks` pages: the `first` first ones, the `recent` last
 * ones up to P, and of those between the ones whose score
 *     max over the KV head's query heads of sum_d max(q_d low_d, q_d high_d)
 * is largest, an upper bound of the products of the page's keys with its queries; equal
 * scores go to the lower page, and a page without a page id in the pool is lowest. The
 * choice is that of sums in 64 bits, so of exact arithmetic unless two scores agree to
 * some 15 digits; with a non-finite query or bound it is unspecified (still `blocks`
 * pages of the sequence). blocks >= first + recent,
 * first >= 0, recent >= 1, blocks <= 8192; sequences of more than 16384 pages are
 * reported as bad extents (4) and left out. selected may be NULL; else it is
 * [rows][kvheads][blocks] and gets the pages of every new row in ascending order, -1
 * behind the last (rows at negative places: -1). Contract, limits and precision as
 * gpu_paged_attention (bounds of pages below P must be up to date: a stale or wild one
 * changes the choice, nothing else). The handle's scratch holds the tables of as many
 * rows as fit 64 MB, four at least; more rows go in turns. */
int gpu_paged_sparse_attention(TcmGpu *, float *out, long long out_stride, const float *q, long long q_stride,
                               const TcmPagedCache *, const TcmPagedBatch *, const uint16_t *bounds, int qheads, int blocks,
                               int first, int recent, int *selected, int *status);

/* ---- Sampling (no counterpart in the reference; gpu_top2 is the greedy readout) ----
 * Each row's settings, in device memory: temperature >= 0 (0: the largest logit, the
 * lowest id among equals), top_k (<= 0: off), top_p (>= 1: off), min_p (<= 0: off). */
typedef struct {
    float temperature;
    int top_k;
    float top_p, min_p;
} TcmSampling;
/* Draw one token a row: logits[r * stride .. + vocab), FP32, -infinity for tokens that
 * may not come. With w_i = exp((logit_i - largest) / temperature) and tokens ranked by
 * logit, equal ones by lower id, kept is the least of: the top_k first; of those, the
 * fewest first ones whose w add up to top_p of theirs or more (one at least); those with
 * w >= min_p. The token is the first kept one, by id, at which the sum of the kept w
 * passes uniforms[r] in [0, 1) times their whole sum. ids, logprobs (the log of the
 * token's share of that sum) and kept (how many are) are [rows]; logprobs and kept may
 * be NULL. stride >= vocab, or 0: every row draws from the same logits. vocab is 1 to
 * 524288. Weights are off by 2^-30 of themselves or 2^-44 of the largest at most, and
 * added exactly, so the same call gives the same tokens. A row that has no
 * token gets id -1, logprob 0, kept 0, and a bit of *status (as above; may be NULL): 1 a
 * logit is NaN or +infinity, 2 no logit is above -infinity, 4 its settings or its uniform
 * are out of range. Returns 0 when launched, or -1 with a message on stderr. */
int gpu_sample(TcmGpu *, int *ids, float *logprobs, int *kept, const float *logits, long long stride, int rows, int vocab,
               const TcmSampling *params, const float *uniforms, int *status);

#ifdef __cplusplus
}
#endif
#endif
