// logits_edit.cu — penalties for repeated tokens, biases and masks on logits, and the greedy choice, in one launch.
//
// A row is read and written once: 2 x 2 or 2 x 4 bytes per logit, its history once per segment from L2. Of a segment of tokens a CTA
// keeps one word each in shared memory: whether the prompt holds the token, how often the rest of the history does, and the first
// bias entry that names it. The counts are whole numbers added by atomics, so their order does not matter; biases of the same token
// are summed in the order of their list. A cluster of up to 8 CTAs shares a row when there are few rows; the choice is the
// maximum of (value, inverted token) keys, which no order changes either.
//
// Rows may start anywhere: a row is cut at the 16-byte boundaries of its input; the vectors at its ends are taken element by
// element, and so are stores to an output that is aligned otherwise.
#include <algorithm>

#include "linear.cuh"
#include "logits_edit.cuh"
#include "ptx.cuh"

namespace b200 {
namespace edit {
namespace {

constexpr int NT = 512;
constexpr int SEG = 16384;  // tokens of a segment: 64 KB of words
constexpr int MAX_CLUSTER = 8;
constexpr int BATCH = 2;  // vectors per thread in flight

// A token's word: bit 31 in the prompt; bits 20..30 MAX_BIAS - i of its first bias entry i (0: none); below, how often it occurs behind
// the prompt.
constexpr uint32_t SEEN = 1u << 31;
constexpr int BIAS_AT = 20;
constexpr uint32_t COUNT = (1u << BIAS_AT) - 1;
constexpr int MAX_BIAS = 1024;          // entries of a row's list
constexpr int MAX_HISTORY = COUNT;      // tokens of a row's history

struct Params {
    void *out;
    const void *in;
    long long ldo, ld;
    int V, cluster;
    int seg;      // tokens per segment
    int len_add;  // added to every length (the decoder's positions)
    int in_place;
    GPT2LogitsEdit e;
    int *next;
    unsigned *status;
};

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(float v, __half &h) { h = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, float &h) { h = v; }

// The largest of a vector's values, NaN left out (-inf if there is nothing else).
__device__ __forceinline__ float top_of(const uint4 &v, __half) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&v);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float top_of(const uint4 &v, float) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}

__device__ __forceinline__ int clamped(int v, int lo, int hi, bool tell, unsigned *status) {
    if (v >= lo && v <= hi) return v;
    if (tell) atomicOr(status, ST_EDIT_BAD_INPUT);
    return min(max(v, lo), hi);
}

struct Row {  // what a row's edits need
    float rep, freq, pres;
    int nb;
    const int *btok;    // shared memory
    const float *bval;  // shared memory
    const int *dups;    // shared memory: some token has several biases
};

__device__ __forceinline__ float edited(float x, uint32_t word, const Row &r) {
    const uint32_t c = word & COUNT, f = word >> BIAS_AT & (2 * MAX_BIAS - 1);
    if (c || (word & SEEN)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, static_cast<float>(c))), r.pres);
    if (f) {
        const int i = MAX_BIAS - static_cast<int>(f);
        float sum = r.bval[i];
        if (*r.dups)
            for (int j = i + 1; j < r.nb; ++j)
                if (r.btok[j] == r.btok[i]) sum += r.bval[j];
        x = __fadd_rn(x, sum);
    }
    return x;
}

template <typename T>
__global__ void __launch_bounds__(NT) k_logits_edit(const Params p) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(16) uint32_t words[];  // a segment's words, the bias list behind them
    __shared__ unsigned long long best[NT / 32], row_best[MAX_CLUSTER];
    __shared__ int dups;
    const long long row = blockIdx.x / p.cluster;
    const int rank = static_cast<int>(blockIdx.x % p.cluster);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const GPT2LogitsEdit &e = p.e;
    int *btok = reinterpret_cast<int *>(words + p.seg);
    float *bval = reinterpret_cast<float *>(btok + e.max_bias);
    if (p.cluster > 1) cluster_arrive_relaxed();  // waited for before the first write to another CTA
    for (int i = tid; i < p.seg / 4; i += NT) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dups = 0;
    grid_dependency_wait();

    const T *in = static_cast<const T *>(p.in) + row * p.ld;
    T *out = static_cast<T *>(p.out) + row * p.ldo;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));  // elements from the boundary to the row
    const bool same = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const bool lean = p.in_place && !p.next;  // vectors without an edit stay where they are, unread
    const bool tell = tid == 0 && rank == 0;

    int n = 0, from = 0;
    const int *hist = nullptr;
    if (e.history && e.max_history > 0) {
        hist = e.history + row * e.history_stride;
        n = clamped(e.length ? e.length[row] + p.len_add : e.max_history, 0, e.max_history, tell, p.status);
        if (e.prompt) from = clamped(e.prompt[row], 0, n, tell, p.status);
    }
    Row r;
    r.rep = e.repetition ? e.repetition[row] : 1.0f;
    r.freq = e.frequency ? e.frequency[row] : 0.0f;
    r.pres = e.presence ? e.presence[row] : 0.0f;
    r.nb = 0;
    r.btok = btok;
    r.bval = bval;
    r.dups = &dups;
    if (e.bias_token && e.max_bias > 0) {
        r.nb = e.n_bias ? clamped(e.n_bias[row], 0, e.max_bias, tell, p.status) : e.max_bias;
        for (int i = tid; i < r.nb; i += NT) {
            btok[i] = e.bias_token[row * e.bias_stride + i];
            bval[i] = e.bias[row * e.bias_stride + i];
        }
    }
    const unsigned *mask = nullptr;
    const int mask_words = (p.V + 31) / 32;
    if (e.mask) {
        int m = e.mask_row ? e.mask_row[row] : e.mask_rows == 1 ? 0 : static_cast<int>(row);
        if (m < -1 || m >= e.mask_rows) {
            if (tell) atomicOr(p.status, ST_EDIT_BAD_INPUT);
            m = -1;
        }
        if (m >= 0) mask = e.mask + m * e.mask_stride;
    }

    float top = -INFINITY;
    int at = -1;
    const int vectors = (p.V + shift + VEC - 1) / VEC, per = (vectors + p.cluster - 1) / p.cluster;
    const int v1 = min(vectors, (rank + 1) * per);
    for (int base = rank * per; base < v1; base += p.seg / VEC) {
        const int m = min(p.seg / VEC, v1 - base);
        const int t0 = base * VEC - shift;  // the token of the segment's first word: below 0 in a row's first vector
        const auto whole = [&](int v) { return t0 + v * VEC >= 0 && t0 + v * VEC + VEC <= p.V; };
        uint4 x[BATCH];
        const auto fetch = [&](int v) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (v + j * NT < m && whole(v + j * NT)) x[j] = *reinterpret_cast<const uint4 *>(in + t0 + (v + j * NT) * VEC);
        };
        if (!lean) fetch(tid);  // on its way while the history is counted
        __syncthreads();
        for (int i = tid; i < r.nb; i += NT) {
            const int t = btok[i];
            if (t >= 0 && t < p.V && static_cast<unsigned>(t - t0) < static_cast<unsigned>(m * VEC))
                if (atomicMax(&words[t - t0], static_cast<uint32_t>(MAX_BIAS - i) << BIAS_AT)) dups = 1;
        }
        if (r.nb) __syncthreads();  // the counts below go under the entries
        for (int i = tid; i < n; i += NT) {
            const int t = hist[i];
            if (t >= 0 && t < p.V && static_cast<unsigned>(t - t0) < static_cast<unsigned>(m * VEC)) {
                if (i < from)
                    atomicOr(&words[t - t0], SEEN);
                else
                    atomicAdd(&words[t - t0], 1u);
            }
        }
        __syncthreads();
        for (int v = tid; v < m; v += NT * BATCH) {
            if (v != tid && !lean) fetch(v);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int u = v + j * NT;
                if (u >= m) break;
                const int t = t0 + u * VEC;
                uint32_t w[VEC], any = 0;
#pragma unroll
                for (int i = 0; i < VEC; i += 4) {
                    const uint4 q = *reinterpret_cast<const uint4 *>(words + u * VEC + i);
                    w[i] = q.x;
                    w[i + 1] = q.y;
                    w[i + 2] = q.z;
                    w[i + 3] = q.w;
                    any |= q.x | q.y | q.z | q.w;
                }
                if (any) {
#pragma unroll
                    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<uint4 *>(words + u * VEC + i) = make_uint4(0, 0, 0, 0);
                }
                if (!whole(u)) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        if (t + i < 0 || t + i >= p.V) continue;
                        const bool masked = mask && !(mask[(t + i) >> 5] >> ((t + i) & 31) & 1);
                        T h = in[t + i];
                        if (w[i]) from_f(edited(to_f(h), w[i], r), h);
                        if (masked) from_f(-INFINITY, h);
                        if (w[i] || masked || !p.in_place) out[t + i] = h;
                        if (to_f(h) > top) {
                            top = to_f(h);
                            at = t + i;
                        }
                    }
                    continue;
                }
                uint32_t allowed = (1u << VEC) - 1;
                if (mask) {
                    const int k = t >> 5, s = t & 31;
                    const unsigned lo = mask[k], hi = s > 32 - VEC && k + 1 < mask_words ? mask[k + 1] : 0u;
                    allowed &= __funnelshift_r(lo, hi, s);
                }
                const bool changed = any || allowed != (1u << VEC) - 1;
                if (lean) {
                    if (!changed) continue;
                    x[j] = *reinterpret_cast<const uint4 *>(in + t);
                }
                T *h = reinterpret_cast<T *>(&x[j]);
                if (changed) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        if (w[i]) from_f(edited(to_f(h[i]), w[i], r), h[i]);
                        if (!(allowed >> i & 1)) from_f(-INFINITY, h[i]);
                    }
                }
                if (same) {
                    if (changed || !p.in_place) *reinterpret_cast<uint4 *>(out + t) = x[j];
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) out[t + i] = h[i];
                }
                if (p.next && top_of(x[j], T()) > top) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (to_f(h[i]) > top) {
                            top = to_f(h[i]);
                            at = t + i;
                        }
                }
            }
        }
    }
    __syncwarp();
    if (p.cluster > 1) cluster_wait();
    if (p.next) {
        // 0.0 + top: equal zeros have equal keys
        unsigned long long key = at < 0 ? 0ull : lin::argmax_key(top + 0.0f, static_cast<unsigned>(at));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
        if (lane == 0) best[warp] = key;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int i = 1; i < NT / 32; ++i) key = max(key, best[i]);
            if (rank == 0)
                row_best[0] = key;
            else
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(smem_u32(&row_best[rank]), 0)), "l"(key) : "memory");
        }
    }
    __syncwarp();
    if (p.cluster > 1) cluster_sync_all();
    if (p.next && tell) {
        unsigned long long key = row_best[0];
        for (int i = 1; i < p.cluster; ++i) key = max(key, row_best[i]);
        if (!key) atomicOr(p.status, ST_EDIT_NO_TOKEN);
        p.next[row] = key ? lin::argmax_key_index(key) : -1;
    }
}

template <typename T>
int set_attr() {
    return cudaFuncSetAttribute(k_logits_edit<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (SEG + 2 * MAX_BIAS) * 4) == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace

int check(const GPT2LogitsEdit *e, int rows, int V) {
    if (!e || rows < 1 || V < 1 || V > (1 << 30)) return GPT2_B200_EINVAL;
    for (const void *q : {static_cast<const void *>(e->repetition), static_cast<const void *>(e->frequency), static_cast<const void *>(e->presence),
                          static_cast<const void *>(e->history), static_cast<const void *>(e->length), static_cast<const void *>(e->prompt),
                          static_cast<const void *>(e->bias_token), static_cast<const void *>(e->bias), static_cast<const void *>(e->n_bias),
                          static_cast<const void *>(e->mask), static_cast<const void *>(e->mask_row)})
        if (reinterpret_cast<uintptr_t>(q) & 3) return GPT2_B200_EINVAL;
    if (e->max_history < 0 || e->max_history > MAX_HISTORY || e->max_bias < 0 || e->max_bias > MAX_BIAS) return GPT2_B200_EINVAL;
    if (e->history && (e->history_stride < 0 || (e->history_stride && e->history_stride < e->max_history))) return GPT2_B200_EINVAL;
    if (e->bias_token && (!e->bias || e->bias_stride < 0 || (e->bias_stride && e->bias_stride < e->max_bias))) return GPT2_B200_EINVAL;
    if (e->mask && (e->mask_rows < 1 || e->mask_stride < (V + 31) / 32 || (!e->mask_row && e->mask_rows != 1 && e->mask_rows < rows))) return GPT2_B200_EINVAL;
    return GPT2_B200_OK;
}

int prepare(DeviceContext *ctx) {
    if (ctx->edit_attr_done) return GPT2_B200_OK;
    RelaxedCapture relaxed;
    if (set_attr<__half>() != GPT2_B200_OK || set_attr<float>() != GPT2_B200_OK) return GPT2_B200_ECUDA;
    ctx->edit_attr_done = true;
    return GPT2_B200_OK;
}

int launch(DeviceContext *ctx, void *out, long long ldo, const void *in, long long ld, int type, int rows, int V, const GPT2LogitsEdit &e, int len_add, int *next,
           bool pdl, cudaStream_t stream) {
    const int rc = prepare(ctx);
    if (rc != GPT2_B200_OK) return rc;
    const int vec = type == GPT2_BEAM_HALF ? 8 : 4;
    Params p = {};
    p.out = out;
    p.in = in;
    p.ldo = ldo;
    p.ld = ld;
    p.V = V;
    p.e = e;
    if (!e.bias_token) p.e.max_bias = 0;
    p.len_add = len_add;
    p.in_place = out == in;
    p.next = next;
    p.status = ctx->status;
    const long long vectors = (V + 2ll * (vec - 1)) / vec;
    int c = MAX_CLUSTER;
    while (c > 1 && (static_cast<long long>(rows) * c > 4ll * ctx->num_sms || vectors < c * 64)) c /= 2;
    p.cluster = c;
    p.seg = static_cast<int>(std::min<long long>(SEG, (vectors + c - 1) / c * vec));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * c, 1, 1);
    cfg.blockDim = dim3(NT, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.seg + 2 * p.e.max_bias) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (c > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = static_cast<unsigned>(c);
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    if (pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t err = type == GPT2_BEAM_HALF ? cudaLaunchKernelEx(&cfg, k_logits_edit<__half>, p) : cudaLaunchKernelEx(&cfg, k_logits_edit<float>, p);
    return err == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace edit
}  // namespace b200

using namespace b200;

extern "C" int gpt2_logits_edit_b200(void *out, long long ldo, const void *logits, long long ld, int type, int rows, int V, const GPT2LogitsEdit *e, int *d_next,
                                     cudaStream_t stream) {
    const size_t size = type == GPT2_BEAM_HALF ? 2 : 4;
    if ((type != GPT2_BEAM_HALF && type != GPT2_BEAM_FLOAT) || !out || !logits || ld < V || ldo < V || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(logits) % size || (out == logits && ldo != ld) || (reinterpret_cast<uintptr_t>(d_next) & 3) || rows > 0x7FFFFFFF / edit::MAX_CLUSTER)
        return GPT2_B200_EINVAL;
    const int rc = edit::check(e, rows, V);
    if (rc != GPT2_B200_OK) return rc;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    return edit::launch(ctx, out, ldo, logits, ld, type, rows, V, *e, 0, d_next, false, stream);
}
