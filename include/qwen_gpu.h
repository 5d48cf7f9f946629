/* qwen_gpu: C ABI of the MI355X (gfx950) Qwen3-0.6B FP16 engine.
 *
 * Drop-in boundary for the reference's native engine API, qwen_cpu::Model
 * (engine/core.hpp:8-56), exported as plain C: opaque handle, plain pointers
 * and sizes, integer status codes, no exceptions and no C++/torch types.
 * Every function returns QWEN_GPU_OK (0) on success; on failure it returns
 * QWEN_GPU_ERROR and qwen_gpu_last_error() (per calling thread) holds the
 * message, using the reference's wording (engine/core.cpp:235-276, 707-752).
 * One caller at a time per model (engine/core.hpp:23).
 *
 * Decode kernels hand values between the workgroups of one launch, so a
 * launch needs the whole GPU (all 256 CUs) to itself. Calls that run them on
 * models stepped from different threads of one process take a process-wide
 * lock and run one after another; another process decoding on the same GPU
 * at the same time can make a step fail with "Decode step stalled" (a
 * bounded wait that gave up, never a hang).
 *
 * A prefill, step or batched step that fails after validation (a stalled
 * exchange, a HIP error) returns each model to its position before the call,
 * without current logits; K/V rows from that position on are rewritten by
 * the next call. A failed verification resets the model
 * (engine/core.cpp:740).
 */
#ifndef QWEN_GPU_H
#define QWEN_GPU_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QWEN_GPU_OK 0
#define QWEN_GPU_ERROR 1
#define QWEN_GPU_VOCABULARY 151936          /* qwen_cpu::vocabulary, engine/core.hpp:9 */
#define QWEN_GPU_HIDDEN 1024
#define QWEN_GPU_PREFIX_REUSE_CHUNK 512     /* qwen_cpu::prefix_reuse_chunk, engine/core.hpp:10 */

typedef struct qwen_gpu_model qwen_gpu_model;

/* qwen_cpu::Options (engine/core.hpp:11-15). Thread counts are validated
 * (1..64) and echoed; context is 1..4096. */
typedef struct qwen_gpu_options {
    int decode_threads;
    int prefill_threads;
    int context;
} qwen_gpu_options;

/* Message of the last failed call on this thread ("" if none). */
const char* qwen_gpu_last_error(void);

/* qwen_cpu::Model::Model(weights_file, Options), engine/core.hpp:28 and
 * engine/core.cpp:235-290: maps and validates the QWCPU01 pack, then uploads
 * it to GPU 0. options == NULL means {12, 6, 4096}. */
int qwen_gpu_create(const char* weights, const qwen_gpu_options* options, qwen_gpu_model** out);
/* qwen_cpu::Model::~Model, engine/core.hpp:29. NULL is ignored. */
void qwen_gpu_destroy(qwen_gpu_model* model);

/* A further model on the device weights already uploaded for `owner` (no
 * second upload): its own K/V cache, position and buffers. options == NULL
 * copies owner's. The weights stay until the last model using them is
 * destroyed. No reference counterpart (the reference is single-stream): it
 * backs the batched decode below for callers serving several sequences. */
int qwen_gpu_create_sharing(const qwen_gpu_model* owner, const qwen_gpu_options* options, qwen_gpu_model** out);
/* dst becomes src truncated to `positions`: K/V rows 0..positions-1 copied on
 * the device as src computed them, no current logits. The canonical
 * prefix-reuse rewind (engine/INTERFACE.md:94-103; Model::truncate,
 * engine/core.cpp:722-727) applied to a copy; both models share weights.
 * Fails with "Rewind position out of range" unless 0 <= positions <= src's
 * position. */
int qwen_gpu_copy_prefix(qwen_gpu_model* dst, const qwen_gpu_model* src, int positions);
/* One decode step for each of `count` (1..8) distinct models that share
 * weights: models[i] consumes tokens[i] (Model::step, engine/core.hpp:38),
 * with every projection reading each weight matrix once for all rows (FP16
 * matrix cores, FP32 activations split into FP16 hi + lo, FP32 sums) and an
 * online-softmax attention over position pieces (held to the reference's
 * tolerance gate, not bit-equal to a batch-1 step). Rows that models hold as
 * copies of the same prefix (qwen_gpu_copy_prefix) are read from one of
 * them. Every model is validated (pending verification, capacity, token
 * range) before any runs. Afterwards each model has current logits and
 * qwen_gpu_greedy works as after a step. No reference counterpart. */
int qwen_gpu_step_batch(qwen_gpu_model* const* models, const int* tokens, int count);
/* qwen_gpu_step_batch, then next[i] = qwen_gpu_greedy(models[i]) in the same
 * call (one host round trip per step for a greedy decode loop). Fails as
 * either would; on failure next is unspecified. No reference counterpart. */
int qwen_gpu_step_batch_greedy(qwen_gpu_model* const* models, const int* tokens, int count, int* next);

/* Model::reset, engine/core.hpp:32; engine/core.cpp:718-721. */
int qwen_gpu_reset(qwen_gpu_model* model);
/* Model::truncate(position), engine/core.hpp:35; engine/core.cpp:722-727. */
int qwen_gpu_truncate(qwen_gpu_model* model, int position);
/* Model::prefill(ids), engine/core.hpp:37; engine/core.cpp:727,707-714. */
int qwen_gpu_prefill(qwen_gpu_model* model, const int* ids, size_t count);
/* Model::step(token), engine/core.hpp:38; engine/core.cpp:728. */
int qwen_gpu_step(qwen_gpu_model* model, int token);
/* Model::verify_two(first, second) -> VerificationRows, engine/core.hpp:17-22,43;
 * engine/core.cpp:729-741. Borrowed row-major [2 x 151936] logits and
 * [2 x 1024] hidden, valid until commit/reset/truncate or another mutation. */
int qwen_gpu_verify_two(qwen_gpu_model* model, int first, int second, const float** logits,
                        const float** hidden, int* base_position);
/* Model::commit_verified(count), engine/core.hpp:46; engine/core.cpp:742-752. */
int qwen_gpu_commit_verified(qwen_gpu_model* model, int count);
/* Model::logits(), engine/core.hpp:47; engine/core.cpp:753. Borrowed FP32
 * [151936] valid until the next mutation; *count is 0 when there are none. */
int qwen_gpu_logits(qwen_gpu_model* model, const float** data, size_t* count);
/* Model::hidden(), engine/core.hpp:48-50; engine/core.cpp:754-757. Fails with
 * "No current hidden state" when there are no current logits. */
int qwen_gpu_hidden(qwen_gpu_model* model, const float** data, size_t* count);
/* Model::position(), engine/core.hpp:51. Returns the position (not a status). */
int qwen_gpu_position(const qwen_gpu_model* model);
/* Model::lossless_bf16_cache_bytes(), engine/core.hpp:53; always 0 (engine/core.cpp:759). */
size_t qwen_gpu_lossless_bf16_cache_bytes(const qwen_gpu_model* model);
/* Which batch-1 decode kernels the model runs (no reference counterpart;
 * for tests and benchmarks): 2 one persistent launch per token, 1 two fused
 * launches per layer, 0 separate kernels (no exchanges inside a launch, as
 * when the device does not deal workgroups round-robin over 8 XCDs). */
int qwen_gpu_decode_kernels(const qwen_gpu_model* model);
/* Options actually in effect (echoed by the protocol handshake, engine/main.cpp:71-79). */
int qwen_gpu_get_options(const qwen_gpu_model* model, qwen_gpu_options* options);

/* Greedy Sampler::select of the current logits (engine/main.cpp:51-59):
 * lowest id among maxima, computed on the GPU without copying the logits.
 * Fails with "Nonfinite model logits" or "No current full-vocabulary logits". */
int qwen_gpu_greedy(qwen_gpu_model* model, int* token);
/* Greedy selections of both pending verification rows (engine/main.cpp:138,142). */
int qwen_gpu_verify_greedy(qwen_gpu_model* model, int* first, int* second);
/* verify_two followed by verify_greedy, without copying the rows to host
 * memory: what the protocol's verify-greedy command needs (engine/main.cpp:
 * 128-147 calls verify_two and selects from the returned rows). The rows stay
 * pending for qwen_gpu_commit_verified. No counterpart in the reference class. */
int qwen_gpu_verify_two_greedy(qwen_gpu_model* model, int first, int second, int* first_choice,
                               int* second_choice);

/* Chat-mode candidates of the current logits on the GPU (engine/main.cpp:
 * 51-62: score = (logit - (seen ? 1.5 : 0)) / 0.7, partial sort of the 20
 * best by value descending, id ascending): the k (1..32) best scores
 * (logit - (penalized ? penalty : 0)) / temperature in that order, with their
 * ids. Only these leave the device; the caller draws from them. Fails with
 * "No current full-vocabulary logits" or "Nonfinite model logits" like the
 * reference's select. */
int qwen_gpu_top_scores(qwen_gpu_model* model, float penalty, float temperature, int k, float* values,
                        int* ids);
/* The model's penalized-token flags, the device copy of the sampler's seen
 * set (engine/main.cpp:42,47-49): cleared when `clear` is nonzero, then
 * ids[0..count) set. All flags start clear; reset/truncate leave them as
 * they are (the sampler owns them, as in the reference). */
int qwen_gpu_update_penalized(qwen_gpu_model* model, int clear, const int* ids, size_t count);

/* Synthetic QWCPU01 pack (format: engine/INTERFACE.md:8-21; tensor order of
 * tools/export_native_cpu_weights.py:29-39): matrices N(0, stddev) rounded to
 * FP16 from a counter-based splitmix64 Box-Muller stream, norm gains 1.0.
 * Writes PATH, PATH.index and PATH.manifest.json; refuses existing outputs. */
int qwen_gpu_write_random_pack(const char* path, uint64_t seed, double stddev, int threads);
/* The pack checks of Model::Model without a device: maps PATH and runs the
 * header, index, shape, range, overlap and finiteness checks of
 * engine/core.cpp:235-276 with the same messages (what qwen_gpu_create runs
 * before touching the GPU). For exporters and tools on hosts without one. */
int qwen_gpu_validate_pack(const char* path);

/* Device memory plumbing for callers that hold no other GPU runtime (the
 * op-level entry points below take device pointers). No reference counterpart:
 * they exist so tests and C callers need not load a second HIP runtime. */
int qwen_gpu_device_malloc(size_t bytes, void** pointer);
int qwen_gpu_device_free(void* pointer);
int qwen_gpu_memcpy_to_device(void* device, const void* host, size_t bytes);
int qwen_gpu_memcpy_to_host(void* host, const void* device, size_t bytes);
int qwen_gpu_device_synchronize(void);

/* Kernel-level entry points on caller-owned device memory (stream may be
 * NULL for the default stream); used by parity tests and the GEMV microbench.
 * Converts natural row-major FP16 [rows x cols] to the engine's chain-tiled
 * GEMV layout; second != NULL interleaves two equal-shape matrices by 4 rows. */
int qwen_gpu_op_tile_matrix(const uint16_t* first, const uint16_t* second, uint16_t* dst, int rows, int cols,
                            void* stream);
/* y[r] = dot(x, W[r]) with the reference dot's chain order (engine/core.cpp:119-147),
 * W chain-tiled; cols in {1024, 2048, 3072}; rows a multiple of 16. */
int qwen_gpu_op_gemv(const uint16_t* tiled, const float* x, float* y, int rows, int cols, void* stream);
/* Batched projection of the prefill path (engine/core.cpp:292-294, the
 * cblas_sgemm branch): C[M x N] = A[M x K] . W[N x K]^T, or C += when
 * accumulate != 0. A is FP32 (split exactly into FP16 hi + lo on the matrix
 * cores), W natural row-major FP16; N and K multiples of 64, M >= 1. */
int qwen_gpu_op_gemm(const float* a, const uint16_t* w, float* c, int m, int n, int k, int accumulate,
                     void* stream);
/* qwen_gpu_op_gemm without any device allocation, for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc). No counterpart in the reference. The FP16 operand
 * planes live in a static device array of the library (4 MiB per device,
 * held until the process ends), so m * k may be at most 1048576; larger
 * inputs fail with an error and launch nothing. The call only enqueues work
 * on `stream` (NULL: the default stream) and returns; the caller synchronizes
 * before reading c. Every call on one device shares that array: calls that
 * may overlap on a device (other streams, other threads) race and must be
 * serialized by the caller. Results are bit-identical to qwen_gpu_op_gemm. */
int qwen_gpu_op_gemm_static(const float* a, const uint16_t* w, float* c, int m, int n, int k, int accumulate,
                            void* stream);
/* Gate/up projection of the prefill path with its SwiGLU epilogue
 * (engine/core.cpp:630-639 with batch > 1: the gate and up projections, then
 * gate * sigmoid(gate) * up): w natural FP16 [n x k] holding
 * n / 2 gate rows then n / 2 up rows, a FP32 [m x k]; act[m][i] is written
 * as FP16 hi and lo planes [m x n / 2] and exponents act_exp [m x n / 16]
 * (one byte per group of 8 activations), with
 * act = (hi + lo) * 2^act_exp[m][i / 8] (the FP32 result to 2^-22; the
 * exponent is 0 unless the group's largest magnitude reaches 65504, the
 * FP16 limit). n a multiple of 256, k of 64. Parity-test entry for the
 * kernel the prefill runs between the post-attention norm and the down
 * GEMM. */
int qwen_gpu_op_gemm_swiglu(const float* a, const uint16_t* w, uint16_t* act_hi, uint16_t* act_lo, uint8_t* act_exp,
                            int m, int n, int k, void* stream);
/* The batch-1 decode projections as a step runs them (parity-test entries;
 * all weights in the chain-tiled layout of qwen_gpu_op_tile_matrix):
 * qkv[4096] = W_qkv . RMSNorm(x, norm_weight) with W_qkv = q, k, v rows
 * stacked [4096 x 1024] (engine/core.cpp:384-386: norm, then project_group<3>
 * over q/k/v). */
int qwen_gpu_op_norm_qkv(const uint16_t* tiled, const float* norm_weight, const float* x, float* qkv, void* stream);
/* act[3072] = SwiGLU(W_gate . h, W_up . h), h = RMSNorm(x + the 16 pending
 * per-query-head O partials parts[16][1024], added in the engine's fixed
 * tree order; parts NULL means none), the tiled matrix interleaving gate and
 * up rows 4 by 4 (qwen_gpu_op_tile_matrix with second = up)
 * (engine/core.cpp:625-639: residual, norm, project_group<2>, SwiGLU).
 * raw (NULL to skip, else [6144]) receives the gate and up dot products in
 * that interleaved row order: 8t + i is gate row 4t + i, 8t + 4 + i up row
 * 4t + i (i < 4). */
int qwen_gpu_op_norm_gate_up(const uint16_t* tiled, const float* norm_weight, const float* x, const float* parts,
                             float* act, float* raw, void* stream);
/* x[r] = (x[r] + the pending O partials of row r, NULL for none) +
 * W_down[r] . act, W_down [1024 x 3072] (engine/core.cpp:640-641: project,
 * then the residual add). */
int qwen_gpu_op_down_residual(const uint16_t* tiled, const float* act, const float* parts, float* x, void* stream);
/* The FFN of one layer as the fused decode kernel runs it
 * (engine/core.cpp:625-641, with the down projection split into 8 column
 * slices): xm = x + the 16 O partials parts[16][1024] (fixed tree order);
 * act = SwiGLU(W_gate . h, W_up . h), h = RMSNorm(xm), posted to
 * exchange[3072] as (tag << 32 | FP32 bits); dparts[g][r] = W_down[r][384 g
 * .. 384 g + 383] . act[384 g .. 384 g + 383] (the reference's 8-chain dot
 * over that slice), g < 8. The next layer adds xm + the 8 slices (see
 * qwen_gpu_op_norm_qkv_folded). exchange must hold no word carrying tag
 * (zero it once; tag != 0 and different from the previous call's); *stall
 * is set nonzero if a workgroup gave up waiting for the slice's
 * activations. Parity-test entry. */
int qwen_gpu_op_fused_ffn(const uint16_t* gateup_tiled, const uint16_t* down_tiled, const float* norm_weight,
                          const float* x, const float* parts, float* xm, float* dparts, uint64_t* exchange, int* stall,
                          uint32_t tag, void* stream);
/* qkv[4096] = W_qkv . RMSNorm(x) where x = xm + the 8 down slices
 * dparts[8][1024] added in the fixed tree order ((d0+d1)+(d2+d3)) +
 * ((d4+d5)+(d6+d7)); x[1024] is written out (engine/core.cpp:641 then
 * 384-386). Parity-test entry. */
int qwen_gpu_op_norm_qkv_folded(const uint16_t* tiled, const float* norm_weight, const float* xm,
                                const float* dparts, float* x, float* qkv, void* stream);
/* Causal GQA attention of a prefill chunk (engine/core.cpp:407-605, the
 * batched rows' attention): rows queries at positions pos0 .. pos0 + rows - 1
 * from qkv FP32 [rows x 4096] (columns 0..2047: 16 query heads of 128),
 * against FP16 keys / values [8 KV heads][context][128] holding positions
 * 0 .. pos0 + rows - 1 (query head h reads KV head h / 2; q and k channels in
 * one common order), scale 1/sqrt(128). Output [rows x 2048] as FP16 hi and
 * lo planes (hi + lo is the FP32 result to 2^-22). rows 1..4096, pos0 + rows
 * <= context. Parity-test entry for the kernel the prefill runs between its
 * QKV and O GEMMs. */
int qwen_gpu_op_attention_prefill(const float* qkv, const uint16_t* keys, const uint16_t* values, uint16_t* att_hi,
                                  uint16_t* att_lo, int rows, int pos0, int context, void* stream);
/* Batched projection of the multi-sequence decode: y[b] = W x[b] for b <
 * batch (1..8) on the matrix cores; W natural row-major FP16 [rows x cols],
 * x FP32 [batch x cols], y FP32 [batch x rows]; rows a multiple of 16, cols
 * in {1024, 2048, 3072}. No reference counterpart (parity-test entry). */
int qwen_gpu_op_bgemv(const uint16_t* w, const float* x, float* y, int batch, int rows, int cols, void* stream);
/* Isolated GEMV microbenchmark: average milliseconds of one op_gemv launch
 * over `iterations` back-to-back launches on the default stream, timed with
 * HIP events, cycling through `copies` chain-tiled weight copies laid
 * `copy_stride` bytes apart (enough copies keep the weights streaming from
 * HBM rather than the 256 MB Infinity Cache). No reference counterpart. */
int qwen_gpu_op_gemv_time(const uint16_t* tiled, size_t copy_stride, int copies, const float* x, float* y, int rows,
                          int cols, int iterations, float* milliseconds);
/* Plain 16-byte-per-thread device copy (bytes a multiple of 16). No reference
 * counterpart: a kernel of known traffic for calibrating HBM byte counters. */
int qwen_gpu_op_copy(const void* src, void* dst, size_t bytes, void* stream);
/* ---- Paged key-value cache (no reference counterpart) ----
 *
 * Keys and values of many sequences in pages of `page_size` slots. Sequence
 * s holds its j-th cached row in slot j % page_size of page
 * table[s * table_stride + j / page_size]; sequences may share pages that
 * neither appends to nor evicts from. Element d of kv head h, slot i, page p
 * lies at p * page_stride + h * head_stride + i * slot_stride + d (strides in
 * elements, equal for keys and values, multiples of 16 bytes; both pointers
 * aligned to 16 bytes; rows must not overlap). [page][head][slot][d] and
 * [page][slot][head][d] are two such layouts, and a contiguous
 * [head][position][d] cache is one with page_stride = page_size * head_dim.
 *
 * Everything else is indexed per sequence, so that shared pages share no
 * state: row j of kv head h of sequence s has its accumulated attention
 * weight and its position in the text at [(s * kv_heads + h) * track_stride
 * + j] of `weights` and `positions`.
 *
 * The device reads table, lengths, offsets and seen when the launch runs, so
 * a captured graph follows them. What they hold cannot be checked on the
 * host and is bounded on the device instead: lengths are taken into 0 ..
 * max_length; a slot whose page is not in 0 .. pages - 1 is neither written
 * nor attended; rows outside 0 .. total_rows - 1 are neither read nor
 * written; offsets must not fall (where they do, which of its rows a sequence
 * gets and what its weights grow by are open). None of them may change while a call runs. `stream` is NULL
 * (the default stream of the cache's device) or a created stream of that
 * device; the current device does not matter. */
#define QWEN_GPU_PAGED_F16 0
#define QWEN_GPU_PAGED_BF16 1
#define QWEN_GPU_PAGED_E4M3 2   /* rows of e4m3 * 2^(exponent byte - 127) */

typedef struct qwen_gpu_paged_cache {
    void* keys;
    void* values;
    uint8_t* exponents;         /* E4M3: [pages][kv_heads][page_size][2], of the key row and of the value row,
                                 * bytes 1..254 */
    int64_t page_stride;
    int64_t head_stride;
    int64_t slot_stride;
    int pages;
    int page_size;              /* 1..65536 */
    int kv_heads;               /* 1..1024 */
    int head_dim;               /* 64, 128 or 256 */
    int type;                   /* QWEN_GPU_PAGED_* */
} qwen_gpu_paged_cache;

typedef struct qwen_gpu_paged_batch {
    const int32_t* table;       /* [sequences][table_stride] */
    const int32_t* lengths;     /* [sequences]: cached rows, the new ones among them */
    const int32_t* offsets;     /* [sequences + 1]: new rows offsets[s] .. offsets[s + 1] - 1 are sequence s's, at
                                 * most `rows` of them; NULL: s has rows s * rows .. (s + 1) * rows - 1 */
    const int32_t* seen;        /* [sequences]: tokens of the text so far, evicted ones too; NULL: lengths */
    float* weights;             /* [sequences][kv_heads][track_stride], or NULL: not tracked */
    int32_t* positions;         /* the same */
    int64_t track_stride;       /* at least max_length where one of them is given */
    int sequences;              /* 1..4096 */
    int table_stride;           /* pages in a row of the table */
    int max_length;             /* 1..table_stride * page_size, at most 2^24 */
    int rows;                   /* 1..2^24: most new rows of a sequence */
    int total_rows;             /* new rows of all sequences; sequences * rows where offsets is NULL */
} qwen_gpu_paged_batch;

/* Bytes of workspace (device memory, aligned to 16) that the attention and
 * the eviction of this cache and batch need at most. The caller zeroes its
 * first QWEN_GPU_PAGED_COUNTER_BYTES once; every call leaves it ready for the
 * next, of whatever shape it suffices for. Calls that may overlap need
 * workspaces of their own, and so do captured graphs that may. query_heads 0:
 * what the eviction alone needs, which does not use offsets, rows and
 * total_rows. Of the attention of tracked weights it holds 4 bytes for each
 * new row, query head and position up to max_length: long prompts are best
 * given in parts, whose weights add up. */
#define QWEN_GPU_PAGED_COUNTER_BYTES 131072
int qwen_gpu_op_paged_workspace(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch, int query_heads,
                                size_t* bytes);
/* The new rows' keys and values, FP32, rounded to the cache's type (to
 * nearest, ties to even) in their slots: row i of sequence s's n goes to slot
 * lengths[s] - n + i, a negative one nowhere. Head h of row r lies at keys +
 * r * key_stride + h * head_dim, so a projection's rows are read where they
 * are. E4M3: the exponent is the smallest of -126 .. 127 that brings the
 * row's largest finite magnitude to 448 or below; infinities and NaN become
 * NaN. As any rounding may, that of the largest numbers can pass the type's
 * (FP16 from 65520 on) or FP32's (248 * 2^120 and more in E4M3 become 2^128):
 * attention takes such elements as infinite. Where tracked, the slots'
 * weights are set to 0 and their positions to seen[s] - n + i. No two rows of
 * a call may go to one slot. */
int qwen_gpu_op_paged_append(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch, const float* keys,
                             int64_t key_stride, const float* values, int64_t value_stride, void* stream);
/* Attention of the new rows over the cached ones, which hold the new ones
 * already: query head g of row r (at queries + r * query_stride + g *
 * head_dim, FP32) reads kv head g / (query_heads / kv_heads). Row i of
 * sequence s's n attends slots 0 .. lengths[s] - n + i with softmax(scale *
 * q . k); a row that has none gives zeros. out is laid out like queries, with
 * out_stride. With weights, weights[s][h][j] grows by the sum of slot j's
 * softmax weights over h's query heads and s's new rows. Sums are FP32, in
 * an order that depends on the call's shapes and lengths alone. Keys and
 * values that a row attends are finite (else its output may be NaN); those
 * that it does not attend may be anything. q . k, with and without the scale,
 * and 256 times the sum of the attended values' magnitudes stay below 2^128
 * (an FP16 cache's values do). out may be queries themselves, with one
 * stride, and lies apart from them otherwise. query_heads is at most 1024 *
 * kv_heads; scale, and scale times log2(e), are finite. */
int qwen_gpu_op_paged_attention(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch,
                                const float* queries, int64_t query_stride, int query_heads, float scale, float* out,
                                int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);
/* Cuts every sequence longer than `keep` to `keep` rows, for each kv head by
 * itself: rows at positions below `sinks` or from seen[s] - recent on stay
 * (sinks + recent <= keep), then those of the largest weight, of equal ones
 * the lowest slot (NaN counts as the lowest weight, -0 as 0). The kept rows
 * in slots from keep on move, in their order, into the holes before it, so
 * the rows no longer lie in the order of their positions: attention of the
 * rows that are appended next does not depend on it. new_lengths[s] =
 * min(lengths[s], keep), not the array `lengths` or `seen`; new_weights and
 * new_positions receive the first new_lengths[s] entries and may be the
 * batch's own arrays (else they must not overlap them). weights and
 * positions are needed; offsets, rows and total_rows are not used. The
 * sequences' pages must be their own. */
int qwen_gpu_op_paged_evict(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch, int keep, int sinks,
                            int recent, int32_t* new_lengths, float* new_weights, int32_t* new_positions,
                            void* workspace, size_t workspace_bytes, void* stream);
/* Attention of the new rows, as qwen_gpu_op_paged_attention, for a batch
 * whose sequences share the first positions of their text: each group's
 * prefix is read once for all of its sequences. Group g has the sequences
 * offsets[g] .. offsets[g + 1] - 1 (bounded to 0 .. sequences on the device;
 * offsets must not fall), which hold the same keys and values in their first
 * lengths[g] slots; those are read through the table of its first sequence
 * with new rows. The prefix is taken no longer than what each of the group's
 * sequences with new rows had cached before them, and a sequence of no group
 * has none, so every row attends what qwen_gpu_op_paged_attention gives it.
 * max_length and max_rest size the launch and share the GPU out between the
 * prefixes and what is behind them; what a sequence has beyond them is attended
 * too, by fewer workgroups. Give max_rest what sequences have as a rule, not
 * the most that they may reach, which would leave few workgroups to the prefix:
 * 64 sequences behind 8192 positions with up to 500 more take 42 us with a
 * max_rest of 500, 49 with 128, 408 with 32768. Sizes that come to 2^24
 * workgroups or more, or to 2^24 rows, are refused. Weights are not tracked:
 * batch->weights and batch->positions must be NULL. The workspace (device
 * memory, aligned to 16) needs no zeroing and keeps nothing between calls. A
 * part of the positions takes 4 * head_dim + 8 bytes of it for each new row and
 * query head; it holds one part of the prefixes and one behind them at least,
 * more where few rows leave room on the GPU (tens of MiB), and behind the
 * prefixes as long as all of theirs fit 256 MiB. */
typedef struct qwen_gpu_paged_prefix {
    const int32_t* lengths;     /* [groups] */
    const int32_t* offsets;     /* [groups + 1]; NULL: one group of all sequences */
    int groups;                 /* 1..sequences; 1 where offsets is NULL */
    int max_length;             /* 0..batch->max_length: most positions of a prefix */
    int max_rest;               /* 1..batch->max_length: positions of a sequence behind its prefix, as a rule */
} qwen_gpu_paged_prefix;

int qwen_gpu_op_paged_shared_workspace(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch,
                                       const qwen_gpu_paged_prefix* prefix, int query_heads, size_t* bytes);
int qwen_gpu_op_paged_attention_shared(const qwen_gpu_paged_cache* cache, const qwen_gpu_paged_batch* batch,
                                       const qwen_gpu_paged_prefix* prefix, const float* queries, int64_t query_stride,
                                       int query_heads, float scale, float* out, int64_t out_stride, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* ---- Pages and rows of a step (no reference counterpart) ----
 *
 * Which pages a sequence has, kept on the device: the sequences' tables and a
 * stack of the free pages, free_pages[0 .. free_count[0] - 1]. */
typedef struct qwen_gpu_paged_pool {
    int32_t* table;             /* [sequences][table_stride]; entries from held[s] on may hold anything */
    int32_t* free_pages;        /* [pages] */
    const int32_t* held;        /* [sequences]: pages in a sequence's row of the table */
    const int32_t* free_count;  /* [1] */
    const int32_t* shared;      /* [sequences]: its first pages, which others use too and are never given back; or NULL */
    int pages;                  /* 1..2^30 */
    int page_size;              /* 1..65536 */
    int sequences;              /* 1..4096 */
    int table_stride;           /* 1..2^24 */
} qwen_gpu_paged_pool;

typedef struct qwen_gpu_paged_growth {
    const int32_t* lengths;     /* [sequences]: cached rows */
    const int32_t* seen;        /* [sequences]: tokens of the text, evicted ones too; NULL: lengths, and no new_seen */
    const int32_t* changes;     /* [sequences]: new rows wished for; below zero: cached rows taken back from the end */
    int32_t* new_lengths;       /* [sequences] */
    int32_t* new_seen;          /* [sequences], with seen */
    int32_t* new_held;          /* [sequences] */
    int32_t* new_free_count;    /* [1] */
    int32_t* offsets;           /* [sequences + 1]: as a batch's, of the rows that were granted */
    int32_t* row_sequences;     /* [total_rows] each, or NULL: of every row granted its sequence, */
    int32_t* row_positions;     /*   its position in the text, */
    int64_t* row_slots;         /*   and page * page_size + slot; -1 in all three behind the last row */
    int total_rows;             /* 0..2^24: room for rows */
} qwen_gpu_paged_growth;

/* One step's bookkeeping. First, pages behind the wished lengths are given
 * back: they are pushed on the free stack in the order of the sequences and
 * of their tables. A call with changes of 0 gives back what an eviction has
 * emptied. Then sequences get their new rows, in order: one that needs pages
 * takes them from the stack's end, until one needs more than there are, and
 * from there on only those that need none are granted; and no sequence
 * whose rows, with those granted before, pass total_rows, nor any with new
 * rows behind it. One that is not granted keeps its length and has no rows in `offsets`;
 * one that has fewer pages than the rows it has need takes those too, when it
 * grows.
 * A wish that the table has no entries for (length + change above
 * table_stride * page_size) counts as a change of 0; a change never takes
 * back more than there is. The lengths, seen, held and changes of one call
 * are read before the results are written, so new_lengths may be lengths,
 * new_seen seen, new_held held and new_free_count free_count; otherwise
 * nothing that is written may overlap another array. What the arrays hold is
 * bounded: held into 0 .. table_stride, lengths into 0 .. table_stride *
 * page_size (at most 2^30), free_count into 0 .. pages; pages given back beyond `pages` free ones are dropped. Tables and
 * slots of pages outside 0 .. pages - 1 (which only a wrong stack can hold)
 * get -1 as their slots. Streams as for the paged cache; the device is that
 * of `table`. */
int qwen_gpu_op_paged_reserve(const qwen_gpu_paged_pool* pool, const qwen_gpu_paged_growth* growth, void* stream);

/* ---- Norm and rotation of heads by position (no reference counterpart) ---- */
#define QWEN_GPU_F32 0
#define QWEN_GPU_F16 1
#define QWEN_GPU_BF16 2
#define QWEN_GPU_ROTARY_HALVES 0        /* channel i turns with channel i + dims / 2 */
#define QWEN_GPU_ROTARY_INTERLEAVED 1   /* channel 2 i turns with channel 2 i + 1 */
#define QWEN_GPU_ROTARY_PLAIN 0
#define QWEN_GPU_ROTARY_LINEAR 1
#define QWEN_GPU_ROTARY_BASE 2
#define QWEN_GPU_ROTARY_RAMP 3

typedef struct qwen_gpu_rotary {
    const double* frequencies;  /* device, [dims / 2]: radians a position of pair i; may be NULL where dims is 0 */
    int dims;                   /* even, 0..head_dim: the first channels of a head, which turn */
    int layout;                 /* QWEN_GPU_ROTARY_HALVES or _INTERLEAVED */
    int head_dim;               /* even, 2..512 */
    int type;                   /* QWEN_GPU_F32, _F16 or _BF16: of the rows, read and written */
    float magnitude;            /* the turned channels are multiplied by it: 1, or what scaled positions ask for */
    float epsilon;              /* of the norm, above 0 */
} qwen_gpu_rotary;

/* Heads of a call's rows: channel d of head h of row r lies at r * row_stride
 * + h * head_stride + d (elements; any alignment that the type has). */
typedef struct qwen_gpu_rotary_heads {
    const void* rows;
    void* out;                  /* may be `rows` with its strides; otherwise apart from all heads that are read */
    const float* norm;          /* device, [head_dim]: weights of the RMS norm of each head; NULL: no norm */
    int64_t row_stride;
    int64_t head_stride;
    int64_t out_row_stride;
    int64_t out_head_stride;
    int heads;                  /* 1..4096 */
} qwen_gpu_rotary_heads;

/* Frequencies of `dims` turned channels (host memory, [dims / 2]) and the
 * magnitude (NULL: not wanted) of a rotation with base `base`, f_i =
 * base^(-2 i / dims), scaled for texts `factor` (1 or more) times as long as
 * the `trained` positions:
 * PLAIN   f_i (factor and trained are not used);
 * LINEAR  f_i / factor, positions squeezed;
 * BASE    the base raised to base * factor^(dims / (dims - 2)), which leaves
 *         the first frequency and divides the last by factor;
 * RAMP    f_i where pair i makes `fast` turns or more within the trained
 *         positions, f_i / factor where it makes `slow` or fewer, in between
 *         their mean weighted by where the turns lie between the two;
 *         magnitude 0.1 ln(factor) + 1.
 * The magnitude of the others is 1, and a base that grows past all numbers is
 * refused. RAMP goes by turns. Checkpoints scaled by a ramp over the pairs'
 * indices, between two borders that are rounded to whole pairs, or run with
 * another magnitude, have other frequencies: give qwen_gpu_op_rotate those. */
int qwen_gpu_rotary_frequencies(int scaling, int dims, double base, double factor, double trained, double slow,
                                double fast, double* frequencies, float* magnitude);
/* Every head of every row, normed (x / sqrt(mean x^2 + epsilon) * norm) and
 * its first channels turned by the angle position * frequency: queries and
 * keys (NULL: none) of up to 2^24 rows in one launch. Row r has
 * positions[r] (device); rows of a negative position, such as those behind
 * the last one in a map of qwen_gpu_op_paged_reserve, are neither read nor
 * written. Angles are FP64, the rest FP32, rounded once to the rows' type;
 * the sum of a normed head's squares stays below 2^128.
 * The rotation multiplies (a, b) by magnitude * (cos, sin) as a cos - b sin,
 * b cos + a sin. Streams as for the paged cache; the device is that of
 * queries->out. */
int qwen_gpu_op_rotate(const qwen_gpu_rotary* rotary, const qwen_gpu_rotary_heads* queries,
                       const qwen_gpu_rotary_heads* keys, const int32_t* positions, int rows, void* stream);

/* ---- Verification of drafted tokens (no reference counterpart) ----
 *
 * Sequence s has n rows of logits: row i is the target's for the token behind
 * the row's own, so that row i of the first n - 1 decides on the drafted token
 * tokens[first + i + 1] and the last one is for the token after all drafts. A
 * sequence of one row has no drafts: a token is drawn for it. */
typedef struct qwen_gpu_draft {
    const void* logits;         /* [total_rows] rows of `vocabulary`, logit_stride apart */
    const float* draft;         /* [total_rows] rows of `vocabulary`, draft_stride apart: the probabilities that row
                                 * i's drafted token was drawn from (last rows are not read); NULL: it was certain */
    const int32_t* tokens;      /* [total_rows]: the rows' own tokens */
    const int32_t* offsets;     /* [sequences + 1]: as a paged batch's; NULL: `rows` rows each */
    const float* temperature;   /* [sequences], NULL: 1 */
    const float* accept;        /* [total_rows]: numbers of [0, 1), one for each drafted token, at the row that
                                 * decides on it */
    const float* sample;        /* [sequences]: numbers of [0, 1), for the token that is drawn */
    int64_t logit_stride;       /* elements */
    int64_t draft_stride;
    int type;                   /* of the logits: QWEN_GPU_F32, _F16 or _BF16 */
    int vocabulary;             /* 1..2^24 */
    int sequences;              /* 1..4096 */
    int rows;                   /* 1..1024: most rows of a sequence */
    int total_rows;             /* 0..2^20; sequences * rows where offsets is NULL */
} qwen_gpu_draft;

/* Bytes of workspace (device memory, aligned to 16); it needs no zeroing and keeps nothing between calls. */
int qwen_gpu_op_verify_workspace(const qwen_gpu_draft* draft, size_t* bytes);
/* With p = softmax(logits / temperature) of a row and q its draft's
 * probabilities, the drafted token t is accepted where accept * q(t) < p(t).
 * At the first one that is not, the token is drawn from max(p - q, 0)
 * (from p, where that is 0 throughout), and where all are accepted, from the
 * last row's p: the lowest token up to which the weights' sum passes sample
 * times their whole sum. So the tokens follow the target's distribution
 * whatever the draft's is. Temperatures of 0 and below (and NaN) stand for the
 * limit: the largest logit, of equal ones the lowest token, has all of p.
 * accepted[s] is the number of accepted tokens, next[s] the one drawn, back[s]
 * accepted[s] less the drafted ones, the rows that a paged cache takes back
 * (qwen_gpu_op_paged_reserve's changes); accepted and back may be NULL. What is left out by a
 * filter has a logit of minus infinity; NaN counts as that, an infinite logit
 * as all of p (shared by equal ones). Where a row has no token left, its
 * drafted one is not accepted and next is -1, as it is for a sequence without rows. A drafted
 * token outside the vocabulary is not accepted; probabilities below 0 and NaN
 * count as 0. Weights and sums are FP64, summed in an order that depends on the
 * call's sizes alone. Streams as for the paged cache; the device is that of
 * `logits`. */
int qwen_gpu_op_verify_draft(const qwen_gpu_draft* draft, int32_t* accepted, int32_t* next, int32_t* back,
                             void* workspace, size_t workspace_bytes, void* stream);
/* Average milliseconds of one standalone launch of a decode kernel on the
 * model's stream, timed with HIP events (which: 0 norm+QKV, 1 attention,
 * 2 O, 3 norm+gate/up, 4 down, 5 lm_head, 6 the fused FFN kernel and 7 the
 * fused norm + QKV + attention + O kernel of the two-kernel step, 8 the
 * token kernel that runs all 28 layers of a step in one launch). Needs
 * position() > 0. The O projection runs with the attention (timed as 1: one
 * kernel up to 512 positions, split attention + merge/O beyond) and 2
 * reports 0. Kernels 0-7 replay layer by layer over all 28 layers, 8 replays
 * whole steps. Afterwards the current logits are invalid; timing the
 * attention or the token kernel (1, 7 or 8) also resets the model, so time
 * them last. */
int qwen_gpu_time_kernel(qwen_gpu_model* model, int which, int iterations, float* milliseconds);

#ifdef __cplusplus
}
#endif
#endif
