/* gpt2_b200.h — C ABI of the B200 (sm_100a) causal self-attention library for GPT-2-124M.
 *
 * Drop-in replacements for the attention hot path of MatteoPhan926/bare-metal-gpt2:
 *   prefill : the GPT2Backend.attention slot          (cuda/kernels.cuh:73), implemented by
 *             gpt2_attention_flash in the reference   (cuda/kernels_fused.cu:145-149);
 *   decode  : gpt2_attn_decode over the KV cache      (cuda/kvcache.cuh:54, cuda/kvcache.cu:207-210);
 *   cache   : the GPT2KVCache arena, its alloc/free/reset/step-bytes helpers and the append / prefill
 *             scatter writers (cuda/kvcache.cuh:39-66, cuda/kvcache.cu:25-81,204-206).
 *
 * Conventions (same as the reference unless stated):
 *   - fp16 storage, fp32 accumulation; qkv rows are [q(E) | k(E) | v(E)], head h at h*D in each part;
 *     att rows are E wide. Causal: query i attends keys 0..i; scale 1/sqrt(D).
 *   - The cache layout is the reference's: per layer L, K at data + (2L)*H*maxT*D and V at
 *     data + (2L+1)*H*maxT*D, each [head][pos][dim] (cuda/kvcache.cuh:31-33,61-66).
 *   - All pointers are device pointers unless a parameter says "host". The caller owns every buffer.
 *   - The reference-signature entry points return void and launch on the legacy default stream, as the
 *     reference does; their argument / launch errors are kept in a per-thread "last error"
 *     (gpt2_b200_last_error). The _stream / _status variants return a GPT2_B200_* code.
 *   - Kernels never trap or spin forever: every wait is bounded, and a timeout sets a bit in a
 *     per-device status word read by gpt2_b200_status().
 *   - Shapes: D must be 64 (the reference's flash kernel has the same restriction, kernels_fused.cu:56);
 *     E = H*64; 16-byte aligned qkv / att / cache pointers.
 */
#ifndef GPT2_B200_H
#define GPT2_B200_H

#include <stddef.h>
#include <cuda_runtime_api.h>

#ifdef __cplusplus
#include <cuda_fp16.h>
typedef __half gpt2_half; /* the reference's `half` */
extern "C" {
#else
typedef struct { unsigned short bits; } gpt2_half;
#endif

/* ---------------------------------------------------------------- status codes */
#define GPT2_B200_OK 0
#define GPT2_B200_EINVAL 1      /* bad argument (shape, alignment, length, null pointer) */
#define GPT2_B200_ECUDA 2       /* a CUDA runtime call failed */
#define GPT2_B200_ENOMEM 3      /* allocation refused (cache plan over budget, workspace) */
#define GPT2_B200_EDEVICE 4     /* the device is not compute capability 10.0, or the driver lacks TMA */
#define GPT2_B200_ETIMEOUT 5    /* a kernel's bounded wait expired (see gpt2_b200_status) */
#define GPT2_B200_ECAPTURE 6    /* would need to allocate while the stream is being captured */

/* ---------------------------------------------------------------- the KV cache (reference ABI)
 * Identical layout to GPT2KVCache in cuda/kvcache.cuh:39-44. If the reference's kvcache.cuh is
 * included first, its definition is used (include the reference headers before this one). */
#ifndef GPT2_KVCACHE_CUH
typedef struct GPT2KVCache {
    gpt2_half *data; /* owns the whole arena (device) */
    size_t bytes;
    int maxT, nLayer, nHead, headDim;
    int len;         /* positions currently cached [0, len) */
} GPT2KVCache;
#endif

/* ---------------------------------------------------------------- the backend table (reference ABI)
 * Identical layout to GPT2Backend in cuda/kernels.cuh:68-86 (opaque function pointers here, so this
 * header does not need the reference's weight types). */
#ifndef GPT2_KERNELS_CUH
typedef struct {
    const char *name;
    void (*embed)(void);
    void (*layernorm)(void);
    void (*matmul)(void);
    void (*attention)(gpt2_half *att, const gpt2_half *qkv, int T, int E, int H, int D);
    void (*gelu)(void);
    void (*add)(void);
    void (*matmul_q)(void);
    void (*gemv)(void);
    void (*gemv_q)(void);
} GPT2Backend;

/* fp16 device weights, identical layout to GPT2LayerGPU / GPT2WeightsGPU in cuda/kernels.cuh:19-48
 * (12 layers; every linear weight [out, in] row-major, model/weights.h:3-5). q is the reference's
 * optional INT8 attachment; it is not read here. */
typedef struct {
    gpt2_half *ln1_g, *ln1_b, *qkv_w, *qkv_b, *attn_proj_w, *attn_proj_b,
              *ln2_g, *ln2_b, *fc_w, *fc_b, *proj_w, *proj_b;
} GPT2LayerGPU;
typedef struct {
    gpt2_half *data; /* owns the whole fp16 body (device) */
    size_t n;
    gpt2_half *wte, *wpe; /* wte is also the tied output head */
    GPT2LayerGPU layers[12];
    gpt2_half *lnf_g, *lnf_b;
    const void *q;
} GPT2WeightsGPU;

/* Reusable device activation scratch, identical layout to GPT2ScratchGPU (cuda/kernels.cuh:54). */
typedef struct {
    gpt2_half *x, *ln, *qkv, *att, *ao, *fc, *ff;
    int maxT;
} GPT2ScratchGPU;
#endif

/* ================================================================ prefill attention */

/* Replaces GPT2Backend.attention / gpt2_attention_flash (cuda/kernels.cuh:73,
 * cuda/kernels_fused.cu:145-149): att[T,E] = causal softmax(q k^T / sqrt(D)) v for every head of
 * qkv[T,3E]. Same signature and semantics; runs the tcgen05/TMEM tensor-core kernel on the legacy
 * default stream. */
void gpt2_attention_b200(gpt2_half *att, const gpt2_half *qkv, int T, int E, int H, int D);

/* Stream variant of gpt2_attention_b200 (additive extension; no reference counterpart). */
int gpt2_attention_b200_stream(gpt2_half *att, const gpt2_half *qkv, int T, int E, int H, int D,
                               cudaStream_t stream);

/* Prefill attention that also fills the KV cache: the same att as gpt2_attention_b200, and rows
 * 0..T-1 of layer L of kv (K and V of every head) written exactly as gpt2_kv_scatter_prefill(kv, L,
 * qkv, T) writes them (cuda/kvcache.cu:67-81); rows >= T are left untouched and kv->len is not changed.
 * Replaces the reference's pair of calls in a prefill forward (cuda/forward_cuda.cu:97-98) with one
 * launch: the K/V tiles the attention loads anyway are stored to the cache from shared memory, so K
 * and V are read once. Requires kv->nHead == H and T <= kv->maxT. Additive extension; the reference
 * has no fused counterpart. */
void gpt2_attention_kv_b200(gpt2_half *att, const gpt2_half *qkv, const GPT2KVCache *kv, int L, int T,
                            int E, int H, int D);
int gpt2_attention_kv_b200_stream(gpt2_half *att, const gpt2_half *qkv, const GPT2KVCache *kv, int L,
                                  int T, int E, int H, int D, cudaStream_t stream);

/* Batched prefill: B independent sequences (or layers) in one launch. Sequence b reads
 * qkv + b*qkv_seq_stride and writes att + b*att_seq_stride (strides in elements; 0 = dense,
 * i.e. T*3E and T*E). Additive extension of cuda/kernels.cuh:73 for batch > 1. */
int gpt2_attention_b200_batched(gpt2_half *att, const gpt2_half *qkv, int B, int T, int E, int H,
                                int D, long long qkv_seq_stride, long long att_seq_stride,
                                cudaStream_t stream);

/* ================================================================ decode attention */

/* Replaces gpt2_attn_decode (cuda/kvcache.cuh:54, cuda/kvcache.cu:207-210): M=1 attention of the
 * step's query (the first E halves of qkv) over keys 0..len-1 of layer L of the cache; writes att[E].
 * Split-context flash-decoding with an in-kernel combine. Legacy default stream. */
void gpt2_attn_decode_b200(gpt2_half *att, const gpt2_half *qkv, const GPT2KVCache *kv, int L,
                           int len);

/* Stream variant (additive extension). */
int gpt2_attn_decode_b200_stream(gpt2_half *att, const gpt2_half *qkv, const GPT2KVCache *kv,
                                 int L, int len, cudaStream_t stream);

/* Decode attention for layers L0 .. L0+nL-1 of one cache in ONE launch. Layer l (relative) reads its
 * query at q + l*q_layer_stride and writes att + l*att_layer_stride (elements). The key count is
 * *d_len when d_len is not NULL (a device int, so a captured CUDA graph replays with a growing
 * context), else len. max_len bounds the split count (0 = kv->maxT). Additive extension. */
int gpt2_attn_decode_b200_layers(gpt2_half *att, long long att_layer_stride, const gpt2_half *q,
                                 long long q_layer_stride, const GPT2KVCache *kv, int L0, int nL,
                                 const int *d_len, int len, int max_len, cudaStream_t stream);

/* gpt2_attn_decode_b200_layers with a host length, for callers that must not have the library
 * allocate device memory (a pool allocator that owns all of HBM, a host that freezes allocations
 * after start-up, a latency-critical loop that cannot absorb a synchronising cudaMalloc). No
 * counterpart in the reference. It allocates nothing: its scratch is a fixed ~520 KiB array inside
 * the library image, one per GPU, held until the process exits. It runs k_decode_split (8 threads per
 * key row, split partials merged by the last CTA), not the regular entry point's k_decode_stream;
 * results agree within the library's parity tolerance. Limits: nL * nHead <= 2048 and
 * nL * nHead * ceil(len / 128) <= 1985 (all 12 GPT-2 layers up to 1024 keys); larger requests
 * return GPT2_B200_EINVAL before launching. The first call on a device looks up the array's device
 * address, and under CUDA's lazy module loading that is when the driver places the array in device
 * memory: make the first call on each device during initialisation, before allocations are frozen
 * and before any stream capture. Not valid after cudaDeviceReset. All calls on a device share the
 * array (its counters are cleared at the start of each call): calls that overlap on the GPU race,
 * so keep them ordered. Its status bits are reported by gpt2_b200_status(). */
int gpt2_attn_decode_b200_layers_noalloc(gpt2_half *att, long long att_layer_stride,
                                         const gpt2_half *q, long long q_layer_stride,
                                         const GPT2KVCache *kv, int L0, int nL, int len,
                                         cudaStream_t stream);

/* Decode attention for B independent sequences, one layer each, in ONE launch: sequence b attends
 * over the [H][maxT][D] K and V slabs at k_slabs[b] / v_slabs[b] (device arrays of device pointers)
 * for d_lens[b] keys (device ints), query q + b*q_stride, output att + b*att_stride. max_len bounds
 * the split count. Additive extension (batched decode over a [B] array of caches). */
int gpt2_attn_decode_b200_batched(gpt2_half *att, long long att_stride, const gpt2_half *q,
                                  long long q_stride, const gpt2_half *const *k_slabs,
                                  const gpt2_half *const *v_slabs, const int *d_lens, int B, int H,
                                  int maxT, int max_len, cudaStream_t stream);

/* The attention part of one decode step for every layer (the ordering of
 * gpt2_decode_step_cuda, cuda/kvcache.cu:249-252): append this step's K,V (from qkv rows
 * qkv + l*qkv_layer_stride) at position pos, then attend over len = pos+1 for all layers.
 * pos is *d_pos when d_pos is not NULL (graph replay), else the host value. Two launches.
 * Does not touch kv->len (the reference sets it on the host after the step, kvcache.cu:268). */
int gpt2_b200_decode_attn_step(gpt2_half *att, long long att_layer_stride, const gpt2_half *qkv,
                               long long qkv_layer_stride, GPT2KVCache *kv, const int *d_pos,
                               int pos, cudaStream_t stream);

/* ================================================================ the KV cache */

/* Replaces gpt2_kv_alloc (cuda/kvcache.cu:29-45): one arena of 2*L*H*maxT*D halves for the GPT-2-124M
 * shape (12 layers, 12 heads, D 64), refused (returns 1) when it would leave < 64 MiB free. 0 = ok. */
int gpt2_kv_alloc_b200(GPT2KVCache *kv, int maxT);
/* Same, for an explicit shape (additive extension). */
int gpt2_kv_alloc_shape_b200(GPT2KVCache *kv, int nLayer, int nHead, int headDim, int maxT);
/* Replaces gpt2_kv_free / gpt2_kv_reset / gpt2_kv_step_bytes (cuda/kvcache.cu:47-52). */
void gpt2_kv_free_b200(GPT2KVCache *kv);
void gpt2_kv_reset_b200(GPT2KVCache *kv);
double gpt2_kv_step_bytes_b200(const GPT2KVCache *kv, int len);

/* Replaces gpt2_kv_append_one (cuda/kvcache.cu:57-64,204-206): writes the K and V parts of qkv[3E]
 * into layer L at position pos, 16-byte vector stores. Legacy default stream. */
void gpt2_kv_append_one_b200(GPT2KVCache *kv, int L, const gpt2_half *qkv, int pos);
/* Append for layers L0..L0+nL-1 (rows qkv + l*qkv_layer_stride) on `stream`; position *d_pos if
 * d_pos != NULL (graph replay), else pos. Additive extension of gpt2_kv_append_one. */
int gpt2_kv_append_b200_stream(GPT2KVCache *kv, int L0, int nL, const gpt2_half *qkv,
                               long long qkv_layer_stride, const int *d_pos, int pos,
                               cudaStream_t stream);

/* Replaces gpt2_kv_scatter_prefill (cuda/kvcache.cu:67-81): rows 0..T-1 of qkv[T,3E] into layer L,
 * positions 0..T-1. Legacy default stream. */
void gpt2_kv_scatter_prefill_b200(GPT2KVCache *kv, int L, const gpt2_half *qkv, int T);
int gpt2_kv_scatter_prefill_b200_stream(GPT2KVCache *kv, int L, const gpt2_half *qkv, int T,
                                        cudaStream_t stream);

/* ================================================================ the decode step around attention
 * The reference's decode step (gpt2_decode_step_cuda, cuda/kvcache.cuh:74-76, cuda/kvcache.cu:233-269)
 * runs 135 launches per token for ONE sequence: embed, and per layer LayerNorm, QKV GEMV, K/V append,
 * attention, projection GEMV, add, LayerNorm, FC GEMV, GELU, projection GEMV, add; then the final
 * LayerNorm and the tied-head GEMV. The entry points below run the same step for B sequences at once:
 * every weight matmul is one tcgen05 pass over the weights for all B rows with bias, GELU, residual
 * add and the K/V append fused into its epilogue, the attention is the batched decode kernel above,
 * and the head's epilogue reduces the logits to per-sequence argmax keys. Four weight launches, one
 * attention launch and two LayerNorm launches per layer (87 per step with the embedding, the head and
 * the token bookkeeping). GPT-2-124M shapes only (E 768, 12 layers, 12 heads, vocabulary 50257). */

/* Drop-in for gpt2_decode_step_cuda on the fp16 path: consumes `token` at position `pos` of *kv
 * (kv->len must equal pos), appends every layer's K/V, writes logits[50257] when logits is not NULL
 * and captures the hidden states into caps_blocks when it is not NULL ((12+2)*768 halves: after
 * block L at L*768, final LayerNorm at 12*768, embedding at 13*768 — the reference's layout), then
 * sets kv->len = pos+1. be and s are accepted for signature compatibility and not used: the step's
 * activations live in a plan the library keeps per (weights, cache) pair, allocated by the first
 * call for that pair (about 10 KB plus tensor maps). Legacy default stream; errors go to
 * gpt2_b200_last_error(). */
void gpt2_decode_step_b200(const GPT2Backend *be, const GPT2WeightsGPU *w, GPT2KVCache *kv, int token,
                           int pos, GPT2ScratchGPU *s, gpt2_half *logits, gpt2_half *caps_blocks);

/* A batch of B (1..256) sequences decoded together, sequence b over the cache kvs[b] (host array of
 * B caches in the reference layout, all with the GPT-2-124M shape and the same maxT). Holds its own
 * activations, tensor maps and launch plans; the weights and caches stay owned by the caller. Its calls share the
 * activations: they come from one host thread at a time, on one stream or on streams ordered behind one another. */
typedef struct gpt2_b200_batch gpt2_b200_batch;
int gpt2_b200_batch_create(gpt2_b200_batch **out, const GPT2WeightsGPU *w, const GPT2KVCache *kvs,
                           int B);
/* Releases the batch; synchronises its device first (replays may still be queued). */
void gpt2_b200_batch_destroy(gpt2_b200_batch *bt);

/* One decode step: sequence b consumes d_tokens[b] at position d_pos[b] (device ints), appends its
 * K/V at that position in every layer and attends over d_pos[b]+1 keys. Optional outputs: logits
 * ([B][logits_stride] halves, the fp16 logits) and d_next (B device ints: argmax of each row, the
 * first index on ties). Cache len fields are not touched. */
int gpt2_b200_batch_step(gpt2_b200_batch *bt, const int *d_tokens, const int *d_pos, gpt2_half *logits,
                         long long logits_stride, int *d_next, cudaStream_t stream);

/* Greedy generation in lock-step, one CUDA graph replay per step: at step t (0 <= t < n_steps) every
 * sequence consumes its token at position t; the token for position t+1 is d_prompt[b][t+1] while
 * t+1 < d_plen[b] (the prompt, fed one token per step) and the argmax of step t's logits after that.
 * d_out[b][0..n_steps] receives every sequence's tokens (prompt and generated; out_stride >=
 * n_steps+1). n_steps <= maxT. flags: 0, or GPT2_B200_GEN_ATTENTION_ONLY to replay only the
 * attention launches of each step (same lengths; a timing aid for the attention share). */
#define GPT2_B200_GEN_ATTENTION_ONLY 1
int gpt2_b200_batch_generate(gpt2_b200_batch *bt, const int *d_prompt, long long prompt_stride,
                             const int *d_plen, int n_steps, int *d_out, long long out_stride,
                             int flags, cudaStream_t stream);

/* The batched linear layer the step is built from (additive; the B-row counterpart of the GEMV slot
 * GPT2Backend.gemv / gpt2_gemv_fp16, cuda/kernels.cuh:94, cuda/kvcache.cu:212-214):
 * C[b, n] = epilogue(fp16(sum_k A[b, k] * W[n, k] + bias[n])) for b < B (1..256), W [N, K] row-major,
 * K a multiple of 64, bias may be NULL. epi: GPT2_B200_LINEAR_STORE writes the value, _GELU writes
 * gelu_new of it, _RESID adds it to C (the residual add). 16-byte aligned A and W, lda a multiple
 * of 8 (A's rows are read by TMA), ldc >= N. The plan of a call (tensor maps, split) is cached per
 * host thread for the last 16 argument sets, so a repeated call costs one launch. */
#define GPT2_B200_LINEAR_STORE 0
#define GPT2_B200_LINEAR_GELU 1
#define GPT2_B200_LINEAR_RESID 2
int gpt2_b200_linear(gpt2_half *C, long long ldc, const gpt2_half *A, long long lda,
                     const gpt2_half *W, const gpt2_half *bias, int B, int N, int K, int epi,
                     cudaStream_t stream);
/* The tied-head form: logits[b, n] = fp16(sum_k A[b, k] * W[n, k]) (written when logits is not NULL)
 * and d_next[b] = the first index of the row's maximum. Its per-tile argmax keys live in one buffer
 * per device (grown on demand, never inside a stream capture): calls on one device must not overlap
 * on the GPU. */
int gpt2_b200_linear_argmax(gpt2_half *logits, long long ldl, const gpt2_half *A, long long lda,
                            const gpt2_half *W, int B, int N, int K, int *d_next,
                            cudaStream_t stream);
/* Same signature and meaning as gpt2_gemv_fp16 (the GPT2Backend.gemv slot): C[1, N] = A[1, K] W^T + b,
 * legacy default stream. K must be a multiple of 64 (all GPT-2 weight matmuls). */
void gpt2_gemv_b200(gpt2_half *C, const gpt2_half *A, const gpt2_half *W, const gpt2_half *bias, int N,
                    int K);

/* Kernel launches one gpt2_b200_batch_step / one generate step makes (launch accounting). */
int gpt2_b200_batch_launches_per_step(const gpt2_b200_batch *bt, int flags);

/* ================================================================ beam search over a paged 8-bit cache
 * Additive extension (the reference decodes one sequence greedily over one fp16 arena). Sequences, or
 * the beams of a search, hold their K/V in pages of `page` positions that rows can share:
 *   data  : codes, [nPages][nLayer][K|V][nHead][page][headDim] bytes, so one page of all layers is one
 *           contiguous run;
 *   scale : fp32, [nPages][nLayer][K|V][nHead][page/block], one per block of `block` positions and head:
 *           value = code * scale. kind GPT2_KV8_INT8: codes -127..127; GPT2_KV8_E4M3: e4m3 codes, at
 *           most 448 in magnitude;
 *   table : [nRow][maxPages], the page of positions i*page .. i*page + page-1 of each row, -1 = none;
 *   len   : [nRow], positions held;
 *   ref   : [nPages], how many table entries name the page (0 = free). A caller that pins pages adds
 *           its own holds here.
 *   work  : scratch of at least gpt2_kv8_work_bytes_b200, zeroed once by the owner (gpt2_kv8_alloc_b200 and
 *           _reset_b200 do); the calls leave its counters at zero.
 * All six are device pointers, data / scale / ref / table / len / work 16-byte aligned. headDim is 64 or 128, page and
 * block are 16, 32, 64 or 128 with block <= page, nRow 1..1024. The calls read and write this state and
 * its work area, so calls on one cache must be ordered on the GPU (one stream, or events); calls on
 * different caches are independent. No call allocates or synchronises, so all may be captured.
 * What the device finds wrong (a length outside the table, an entry that is no page, no free page, a
 * parent outside -1..nRow-1, a K/V value or logit that is not finite) sets bits of gpt2_b200_status(). */
#define GPT2_KV8_INT8 0
#define GPT2_KV8_E4M3 1
typedef struct {
    void *data;
    float *scale;
    int *ref, *table, *len;
    void *work;
    size_t work_bytes;
    int nPages, nRow, maxPages, nLayer, nHead, headDim, page, block, kind;
} GPT2KV8Cache;

/* Scratch bytes of a cache of this shape whose gpt2_kv8_attend_b200 calls have at most Hq query heads and
 * Tq queries per row (0 for a bad shape; the pointers are not looked at). */
size_t gpt2_kv8_work_bytes_b200(const GPT2KV8Cache *kv, int Hq, int Tq);
/* Allocates all six arrays for the shape fields set in *kv, as gpt2_kv_alloc_b200 does (refused, 1, when
 * < 64 MiB would stay free; 0 = ok), and resets the cache. */
int gpt2_kv8_alloc_b200(GPT2KV8Cache *kv, int Hq, int Tq);
void gpt2_kv8_free_b200(GPT2KV8Cache *kv);
/* Every page free, every row empty, work area zeroed. */
int gpt2_kv8_reset_b200(const GPT2KV8Cache *kv, cudaStream_t stream);

/* Writes K and V rows of layers L0 .. L0+nL-1 behind the positions each row holds: row r, token t <
 * count_r, goes to position len[r] + t, from k + l*layer_stride + r*row_stride + t*tok_stride (halves; v
 * likewise; head h at h*headDim), where count_r = min(d_count[r], T) if d_count, else T. The pages must be there
 * (gpt2_kv8_reorder_b200's reserve). A block's scale s becomes max(s_old, amax/qmax) (s_old if the block
 * held positions before), the codes round(x * (1/s)) to nearest even; where s grew, the block's older codes become
 * round(code * (s_old/s)). NaN is stored as 0, infinities as the largest fp16 (status bit). len is not
 * changed: gpt2_kv8_reorder_b200's advance counts the tokens in once all layers have stored them. */
int gpt2_kv8_store_b200(const GPT2KV8Cache *kv, int L0, int nL, const gpt2_half *k, const gpt2_half *v,
                        long long layer_stride, long long row_stride, long long tok_stride,
                        const int *d_count, int T, cudaStream_t stream);
/* Reads positions first_r .. first_r + T-1 of each row back as fp16 (code * scale, rounded once), to the
 * same kind of rows; first_r = d_first[r], 0 without d_first. Positions outside 0 .. len[r] + count_r - 1
 * (stored but not yet counted in: count_r = d_count[r], or count) give 0. */
int gpt2_kv8_load_b200(const GPT2KV8Cache *kv, int L0, int nL, gpt2_half *k, gpt2_half *v,
                       long long layer_stride, long long row_stride, long long tok_stride,
                       const int *d_first, int T, const int *d_count, int count, cudaStream_t stream);

/* Attention over layer L: row r has n = len[r] + count_r keys (count_r as above: the tokens stored in this
 * step) and its Tq queries are its last positions n-Tq .. n-1; query i sees keys first_r .. n-Tq+i
 * (d_first NULL: from 0). out = softmax(q K^T / sqrt(headDim)) V, fp32 accumulation, one rounding; a query
 * that sees no key gives 0. (Inside, a probability times its value's scale has 22 bits, or 2^-34 of the row's largest
 * where that is more.) Hq query heads, head h reads K/V head h / (Hq/nHead). q and out: head h at h*headDim, row r at
 * r*row_stride, query t at t*tok_stride (halves, multiples of 8). max_len bounds n (0 =
 * the table's capacity) and sizes the split; a row with n outside 0..max_len sets a status bit and gives 0.
 * With many rows, the leading pages that rows 4 i .. 4 i + 3 (or 2 i, 2 i + 1) all hold are read once for them: keep an item's
 * beams together. Which pages are shared, and max_len, may change the last bit of a result; the same call twice does not. */
int gpt2_kv8_attend_b200(gpt2_half *out, long long out_row_stride, long long out_tok_stride,
                         const gpt2_half *q, long long q_row_stride, long long q_tok_stride,
                         const GPT2KV8Cache *kv, int L, int Hq, int Tq, const int *d_first,
                         const int *d_count, int count, int max_len, cudaStream_t stream);

/* The state behind a selection. First every row counts in `advance` positions; then row r becomes a copy of
 * what row parent[r] held (parent NULL: itself; -1: empty) by holding the same pages; then each row gets room
 * for `reserve` more positions: a partly filled last page that another holder has too is copied to a new
 * page (its filled part), unless this row is the last in row order that is left with it; the missing pages are added.
 * New pages are the lowest-numbered free ones, handed out in row order, a row's copy first. Pages no row holds any more are
 * free. Without enough pages the entry is -1 (status bit). */
int gpt2_kv8_reorder_b200(const GPT2KV8Cache *kv, const int *parent, int advance, int reserve,
                          cudaStream_t stream);
/* Moves the live pages (ref > 0) to the ids 0 .. live-1: the free ids below live, in ascending order, take the live pages
 * at or above it, in ascending order. Tables and ref follow; *d_live (if not NULL) receives the number of live pages. */
int gpt2_kv8_compact_b200(const GPT2KV8Cache *kv, int *d_live, cudaStream_t stream);

/* Beam selection. logits: [B*W][ld] of V values, type GPT2_BEAM_HALF or GPT2_BEAM_FLOAT; score [B*W] the beams' log
 * probabilities so far (-inf: a beam that does not exist, e.g. all but one at the first step); done [B*W] (NULL: none)
 * marks finished beams. Candidate (w, token) of item b has score[w] + logit - logsumexp(row), a finished beam is
 * one candidate (w, eos) with its score unchanged; the W largest per item are chosen, equal totals by the lower w, then the
 * higher logit, then the lower token. -inf logits are masked tokens; NaN and +inf set a status bit and count as masked. Outputs, best first: token,
 * parent (row index b*W + w, as gpt2_kv8_reorder_b200 takes it), new_score, new_done (NULL: not written) = finished
 * before, or token == eos (eos < 0: none). Where fewer than W candidates exist the rest is a dead beam: token max(eos, 0),
 * parent its own row, score -inf, done 1. new_score / new_done may be score / done. W 1..32. work: at least
 * gpt2_beam_work_bytes_b200(B, W) bytes, zeroed once by their owner. One area serves calls of every B and W that it is large enough
 * for; calls that share it must be ordered. */
#define GPT2_BEAM_HALF 0
#define GPT2_BEAM_FLOAT 1
size_t gpt2_beam_work_bytes_b200(int B, int W);
int gpt2_beam_select_b200(int *token, int *parent, float *new_score, int *new_done, const void *logits,
                          int type, long long ld, const float *score, const int *done, int B, int W,
                          int V, int eos, void *work, size_t work_bytes, cudaStream_t stream);

/* Beam search with GPT-2-124M: the decode step of gpt2_b200_batch_step over the 8-bit cache, the selection and the
 * reorder, captured in one CUDA graph. B prompts, W beams each (W 1..32, B*W <= 256), over a cache of B*W rows in the
 * GPT-2-124M shape, whose pages must be enough for what the beams hold apart (status bit otherwise); weights and cache
 * stay owned by the caller. */
typedef struct gpt2_b200_beam gpt2_b200_beam;
int gpt2_b200_beam_create(gpt2_b200_beam **out, const GPT2WeightsGPU *w, const GPT2KV8Cache *kv, int B, int W);
/* Releases the beam decoder; synchronises its device first. */
void gpt2_b200_beam_destroy(gpt2_b200_beam *bm);
/* Empties the cache and runs n_steps steps (at most 1024 and the cache's positions): item b consumes its prompt
 * d_prompt[b][0 .. d_plen[b]-1] one token per step, then its W beams are extended by the W best continuations per step; a
 * beam that chose eos (-1: none) keeps its score and repeats eos. d_out[b*W+w][0..n_steps] receives hypothesis w of item b,
 * best first (prompt included), d_score[b*W+w] (if not NULL) the sum of its chosen tokens' log probabilities. */
int gpt2_b200_beam_generate(gpt2_b200_beam *bm, const int *d_prompt, long long prompt_stride, const int *d_plen, int n_steps,
                            int eos, int *d_out, long long out_stride, float *d_score, cudaStream_t stream);

/* ================================================================ 4-bit weights
 * Additive extension (the reference's own quantised slots, matmul_q and gemv_q of cuda/kernels.cuh:80-85, take 8-bit weights of
 * another form). A weight [N][K] in 4 bits, all arrays on the device and the caller's:
 *   codes : [N][K/2] bytes, 16-byte aligned. Of the 8 elements of a 32-bit word, element 2 i lies in bits 4 i .. 4 i + 3 and
 *           element 2 i + 1 in bits 16 + 4 i .. 16 + 4 i + 3;
 *   scale : [K/group][N], one per `group` (32, 64 or 128) neighbouring k of a row;
 *   least : [K/group][N], or NULL.
 * A code c of 0..15 stands for fp16(c * scale + least), without least for fp16((c - 8) * scale), rounded once. K is a multiple of
 * group, at most 2^24, N at most 2^30; scales and leasts are finite. No call allocates, synchronises or keeps anything of its
 * arguments, so all may be captured. */
typedef struct {
    void *codes;
    gpt2_half *scale, *least;
    int N, K, group;
} GPT2W4;

/* Writes codes, scale and least (if not NULL) for the fp16 weight W (row n at W + n*ldw, 16-byte aligned, ldw a multiple of 8). With least:
 * l = min of the group, s = (max - min) / 15 rounded down to fp16, c = (x - l) * (1 / s) to the nearest, ties to even. Without: s = max|x| / 7
 * rounded down, c = 8 + x * (1 / s) to the nearest, 1..15. s = 0 gives code 0, or 8. NaN counts as 0, infinities as the largest
 * fp16 (status bit). Arithmetic in fp32. */
int gpt2_w4_quantize_b200(const GPT2W4 *w, const gpt2_half *W, long long ldw, cudaStream_t stream);
/* The fp16 values that the codes stand for, to rows of the same kind. */
int gpt2_w4_dequantize_b200(gpt2_half *W, long long ldw, const GPT2W4 *w, cudaStream_t stream);

/* gpt2_b200_linear with a 4-bit weight: C[b, n] = e(sum_k A[b, k] * value(n, k) + bias[n]) for b < B (1..256), sums in fp32, e and one
 * rounding to fp16 behind them: GPT2_B200_LINEAR_STORE the sum, _GELU gelu_new of it, _RESID R[b, n] + the sum (R: rows of stride
 * ldr >= N, may be C itself with ldr = ldc; not read otherwise, may be NULL). bias may be NULL. A 16-byte aligned, lda a multiple of 8, ldc >= N;
 * C must not overlap A, nor R but as said. */
int gpt2_w4_linear_b200(gpt2_half *C, long long ldc, const gpt2_half *A, long long lda, const GPT2W4 *w, const gpt2_half *bias,
                        const gpt2_half *R, long long ldr, int B, int epi, cudaStream_t stream);

/* ================================================================ logits on their way to a choice
 * Penalties for repeated tokens, biases and grammar masks, and the greedy choice, in one pass. All pointers are device pointers
 * and may be NULL where said. Of row r's history the first n = length[r] (NULL: max_history) tokens count, the first prompt[r] (NULL: 0)
 * of them being the prompt. A token t (a token outside 0..V-1 is passed over) with logit x becomes, in fp32 and this order,
 *   x > 0 ? x / repetition[r] : x * repetition[r]    where t is among the n tokens             (repetition NULL: no change)
 *   x - frequency[r] * c - presence[r]               where t is c > 0 times among those behind the prompt (NULL: 0)
 *   x + the sum of bias[r][i] over bias_token[r][i] = t, i < n_bias[r] (NULL: max_bias), in order of i
 *   -inf                                             where the mask's bit of t is 0: bit t % 32 of word t / 32
 * and is rounded once. NaN stays NaN but for masked ones. mask: [mask_rows][mask_stride] words; row r takes row mask_row[r] of it (-1: no
 * mask; mask_row NULL: row r, or the one row there is if mask_rows is 1). Lengths outside 0..max_history, prompts outside 0..n, counts
 * outside 0..max_bias are clamped, a mask row outside -1..mask_rows-1 counts as -1 (status bit). */
typedef struct {
    const float *repetition, *frequency, *presence; /* [rows] */
    const int *history;                             /* [rows][history_stride], NULL: none */
    long long history_stride;
    int max_history; /* 0..2^20 - 1 */
    const int *length, *prompt; /* [rows] */
    const int *bias_token;      /* [rows][bias_stride], NULL: none */
    const float *bias;
    long long bias_stride; /* 0: the same list for all rows; likewise history_stride */
    int max_bias;          /* 0..1024 */
    const int *n_bias;     /* [rows] */
    const unsigned *mask;  /* NULL: none */
    long long mask_stride; /* words, >= ceil(V / 32) */
    int mask_rows;
    const int *mask_row; /* [rows] */
} GPT2LogitsEdit;

/* out[r] = the edited logits[r], r < rows: rows of V values, type GPT2_BEAM_HALF or GPT2_BEAM_FLOAT, at strides ldo and ld >= V
 * (elements; any alignment). out may be logits itself with ldo = ld (then only what changes is written; without a mask and d_next
 * only that is read); otherwise the two must not overlap. d_next (if not NULL): the token of the largest written value of each row, the lowest
 * of equal ones; NaN is never chosen, and a row that has nothing above -inf gives -1 (status bit). */
int gpt2_logits_edit_b200(void *out, long long ldo, const void *logits, long long ld, int type, int rows, int V, const GPT2LogitsEdit *edit,
                          int *d_next, cudaStream_t stream);

/* The decode step over 4-bit weights: gpt2_b200_batch_create with every layer's four matmul weights, and the head's if head.codes is not
 * NULL (else the fp16 wte is the head), in 4 bits: qkv [2304][768], attn_proj [768][768], fc [FFN][768], proj [768][FFN], head
 * [50257][768]. w gives the embeddings, LayerNorms and biases; its matmul weights may be NULL. The 4-bit weights stay owned by the caller.
 * All gpt2_b200_batch_* calls take such a batch. Each output is rounded once, behind bias, GELU or residual. */
typedef struct {
    GPT2W4 qkv[12], attn_proj[12], fc[12], proj[12], head;
} GPT2W4Weights;
int gpt2_b200_batch_create_w4(gpt2_b200_batch **out, const GPT2WeightsGPU *w, const GPT2W4Weights *q, const GPT2KVCache *kvs, int B);

/* gpt2_b200_batch_generate with the logits of every step behind the prompt edited before the choice, in the same graph: sequence b's
 * history is what d_out[b] holds so far, its first d_plen[b] tokens the prompt, so edit's history, length and prompt are NULL; the other
 * arrays have a row per sequence and are the same for all steps of a call, which enqueues them all: work ordered on the stream may change them
 * between calls. (A mask that follows the tokens, a grammar's, needs gpt2_b200_batch_step and gpt2_logits_edit_b200 for each.) A sequence with
 * nothing left to choose gets -1 in d_out (status bits) and goes on from token 0. The first call of a batch allocates its logits. A step
 * makes one launch more than gpt2_b200_batch_launches_per_step says. */
int gpt2_b200_batch_generate_edited(gpt2_b200_batch *bt, const int *d_prompt, long long prompt_stride, const int *d_plen, int n_steps, int *d_out,
                                    long long out_stride, const GPT2LogitsEdit *edit, cudaStream_t stream);

/* ================================================================ backend, status, set-up */

/* Composes a backend the reference's way (cuda/kernels_fused.cu:157-164): copies *base and installs
 * gpt2_attention_b200 as .attention and "b200" as .name. base may be NULL (all other slots NULL). */
void gpt2_b200_compose_backend(GPT2Backend *dst, const GPT2Backend *base);

/* Reserves decode workspace on the current device for `jobs` (layer x sequence) decodes of up to
 * max_len keys, so that later calls (e.g. inside CUDA graph capture) do not allocate. */
int gpt2_b200_reserve(int jobs, int n_head, int max_len);

/* Synchronises the current device and returns the device status word (0 = healthy; bits name the
 * kernel and wait that timed out). clear != 0 resets it. */
unsigned gpt2_b200_status(int clear);

/* Last argument / launch error of a void entry point on this host thread (GPT2_B200_*); clears it. */
int gpt2_b200_last_error(void);
const char *gpt2_b200_strerror(int code);

/* Self-test of the bounded-wait path: launches one CTA that waits on an mbarrier nothing arrives on,
 * with a timeout of timeout_us microseconds. Returns GPT2_B200_ETIMEOUT when the wait expired and the
 * kernel returned cleanly (the expected result); the device context stays usable. */
int gpt2_b200_selftest_wait_timeout(unsigned timeout_us);

/* Library version string. */
const char *gpt2_b200_version(void);

#ifdef __cplusplus
} /* extern "C" */
#endif
#endif /* GPT2_B200_H */
