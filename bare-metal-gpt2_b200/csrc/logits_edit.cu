// logits_edit.cu — penalties for repeated tokens, biases and masks on logits, and the greedy choice, in one launch.
//
// A row is read and written once: 2 x 2 or 2 x 4 bytes per logit. Most logits change by the mask alone, so a CTA works on a segment of
// tokens in two passes: the dense one copies, masks and looks for the largest; the sparse one takes the tokens of the history and of
// the bias list, a few hundred, each once. Between them stands one word per token of the segment in shared memory: whether the
// prompt holds it, how often the rest of the history does, and the first bias entry that names it; a list of the tokens that have one; and
// one bit per token, by which the dense pass leaves those out of the choice. (Edits within the dense pass took 190 instructions per 16 bytes, which cost three times the
// bytes.) The counts are whole numbers added by atomics, so their order does not matter; biases of the same token are summed in
// the order of their list; the choice is the maximum of (value, inverted token), which no order changes either. A cluster of up to 8
// CTAs shares a row when there are few rows.
//
// 256 x 131072 fp32 with 8192 of history, a mask and 300 biases: 89 us (floor 42.7), without any 42.6. The history is looked through by each of a
// row's 8 CTAs, and its tokens' logits are single reads and writes: 30 us. 64 x 50257 fp16 with 1023 of history and a choice: 12.0 us, most of it
// barriers between short passes.
//
// Rows may start anywhere: a row is cut at the 16-byte boundaries of its input; the vectors at its ends are taken element by
// element, and so are stores to an output that is aligned otherwise.
#include <algorithm>
#include <type_traits>

#include "linear.cuh"
#include "logits_edit.cuh"
#include "ptx.cuh"

namespace b200 {
namespace edit {
namespace {

constexpr int NT = 512;
constexpr int SEG = 16384;  // tokens of a segment: 64 KB of words, two CTAs per SM
constexpr int MAX_CLUSTER = 8;
constexpr int BATCH = 4;  // vectors per thread in flight
constexpr int AHEAD = 8;  // tokens of the history per thread in flight

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
    int list;     // touched tokens of a segment at most
    int len_add;  // added to every length; not 0: the decoder's positions, of which those within a prompt are left alone
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

// -inf where a vector's bit is 0.
__device__ __forceinline__ void cut(uint4 &v, uint32_t allowed, __half) {
    uint32_t *w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t keep = (allowed >> (2 * i) & 1) * 0xFFFFu + (allowed >> (2 * i + 1) & 1) * 0xFFFF0000u;
        w[i] = (w[i] & keep) | (0xFC00FC00u & ~keep);
    }
}
__device__ __forceinline__ void cut(uint4 &v, uint32_t allowed, float) {
    uint32_t *w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = allowed >> i & 1 ? w[i] : 0xFF800000u;
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

// One more of a token in the prompt, or behind it; what its word was (1 if neither). Both under predicates: as branches they take three times
// the instructions, and the history is looked at token by token.
__device__ __forceinline__ uint32_t counted(uint32_t word, bool seen, bool count) {
    uint32_t before = 1;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 p, %2, 0;\nsetp.ne.u32 q, %3, 0;\n@p atom.shared.or.b32 %0, [%1], %4;\n@q atom.shared.add.u32 %0, [%1], 1;\n}"
        : "+r"(before)
        : "r"(word), "r"(static_cast<uint32_t>(seen)), "r"(static_cast<uint32_t>(count)), "n"(SEEN)
        : "memory");
    return before;
}

// MASK, NEXT: there is a mask, a choice is asked for.
template <typename T, bool MASK, bool NEXT>
__global__ void __launch_bounds__(NT, 2) k_logits_edit(const Params p) {
    constexpr int VEC = 16 / sizeof(T);
    constexpr uint32_t ALL = (1u << VEC) - 1;
    extern __shared__ __align__(16) uint32_t words[];  // a segment's words, bits, mask and list, the bias list
    __shared__ unsigned long long best[NT / 32], row_best[MAX_CLUSTER];
    __shared__ int dups, n_touched;
    const long long row = blockIdx.x / p.cluster;
    const int rank = static_cast<int>(blockIdx.x % p.cluster);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const GPT2LogitsEdit &e = p.e;
    uint32_t *bits = words + p.seg;         // touched tokens
    uint32_t *allow = bits + p.seg / 32;    // the mask, from the segment's first word on
    uint16_t *touched = reinterpret_cast<uint16_t *>(allow + p.seg / 32);  // in any order: nothing depends on it
    int *btok = reinterpret_cast<int *>(touched + p.list);
    float *bval = reinterpret_cast<float *>(btok + e.max_bias);
    if (NEXT && p.cluster > 1) cluster_arrive_relaxed();  // waited for before the first write to another CTA
    grid_dependency_wait();

    const T *in = static_cast<const T *>(p.in) + row * p.ld;
    T *out = static_cast<T *>(p.out) + row * p.ldo;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));  // elements from the boundary to the row
    const bool same = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const bool tell = tid == 0 && rank == 0;

    int n = 0, from = 0;
    const int *hist = nullptr;
    if (e.history && e.max_history > 0) {
        hist = e.history + row * e.history_stride;
        n = e.length ? e.length[row] + p.len_add : e.max_history;
        if (e.prompt) from = e.prompt[row];
    }
    if (NEXT && p.len_add && n < from) {  // the decoder within a prompt: its next token is there, nothing is chosen or reported
        if (p.cluster > 1) cluster_wait();
        return;
    }
    Row r;
    r.rep = e.repetition ? e.repetition[row] : 1.0f;
    r.freq = e.frequency ? e.frequency[row] : 0.0f;
    r.pres = e.presence ? e.presence[row] : 0.0f;
    r.nb = e.bias_token && e.max_bias > 0 ? (e.n_bias ? e.n_bias[row] : e.max_bias) : 0;
    r.btok = btok;
    r.bval = bval;
    r.dups = &dups;
    const unsigned *mask = nullptr;  // of this row
    if (MASK) {
        int m = e.mask_row ? e.mask_row[row] : e.mask_rows == 1 ? 0 : static_cast<int>(row);
        if (m < -1 || m >= e.mask_rows) {
            if (tell) atomicOr(p.status, ST_EDIT_BAD_INPUT);
            m = -1;
        }
        if (m >= 0) mask = e.mask + m * e.mask_stride;
    }

    // Vector v of a row holds tokens v * VEC - shift .. + VEC - 1; those from f0 to f1 - 1 are whole.
    const int f0 = shift ? 1 : 0, f1 = (p.V + shift) / VEC, vectors = (p.V + shift + VEC - 1) / VEC;
    const int per = (vectors + p.cluster - 1) / p.cluster, v0 = rank * per, v1 = min(vectors, v0 + per), seg = p.seg / VEC;
    // The dense pass has something to do unless the logits stay in place and nothing asks for the mask or the largest.
    const bool dense = MASK || NEXT || !p.in_place;
    n = clamped(n, 0, hist ? e.max_history : 0, tell, p.status);
    from = p.len_add ? min(max(from, 0), n) : clamped(from, 0, n, tell, p.status);
    r.nb = clamped(r.nb, 0, e.max_bias, tell, p.status);
    int h[AHEAD];
    const auto tokens = [&](int i0) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) h[k] = i0 + k * NT + lane < n ? hist[i0 + k * NT + lane] : -1;
    };
    tokens(warp * 32);
    for (int i = tid; i < r.nb; i += NT) {
        btok[i] = e.bias_token[row * e.bias_stride + i];
        bval[i] = e.bias[row * e.bias_stride + i];
    }
    if (n | r.nb)
        for (int i = tid; i < (p.seg + p.seg / 32) / 4; i += NT) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) dups = n_touched = 0;

    float top = -INFINITY;
    int at = -1;
    const auto better = [&](float y, int t) {
        if (y > top || (y == top && at >= 0 && t < at)) {
            top = y;
            at = t;
        }
    };
    for (int base = v0; base < v1; base += seg) {
        const int end = min(base + seg, v1), t0 = base * VEC - shift;  // t0: the token of the first word, below 0 in a row's first vector
        const int lo = max(t0, 0), span = min(end * VEC - shift, p.V) - lo;
        const int d0 = max(base, f0) + tid, d1 = min(end, f1);
        const auto inside = [&](int t) { return static_cast<unsigned>(t - lo) < static_cast<unsigned>(span); };
        if (base != v0) {
            if (n > NT * AHEAD) tokens(warp * 32);
            __syncthreads();  // the words before were read
            if (tid == 0) n_touched = 0;
        }
        if (MASK)
            for (int i = tid; i < p.seg / 32; i += NT) {
                const int t = t0 + i * 32, k = t >> 5, last = (p.V - 1) >> 5;  // k is -1 in front of a row that starts inside a vector
                allow[i] = mask ? __funnelshift_r(k >= 0 ? mask[min(k, last)] : 0u, mask[min(k + 1, last)], t & 31) : 0xFFFFFFFFu;
            }
        const auto masked = [&](int t) { return MASK && !(allow[(t - t0) >> 5] >> ((t - t0) & 31) & 1); };
        __syncthreads();  // the words and the counter are 0, the lists are there

        // The first vectors come while the history is counted. One that is masked whole is not read.
        uint4 x[BATCH];
        uint32_t allowed[BATCH];
        const uint4 *src = reinterpret_cast<const uint4 *>(in - shift);
        const int place32 = (d0 - base) * VEC & 31;  // the same for all vectors of a thread
        const auto fetch = [&](int v, auto whole) {
            const uint32_t *mine = allow + ((v - base) * VEC >> 5);
            const uint4 *sv = src + v;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                if (!whole && v + j * NT >= d1) break;
                if (MASK) allowed[j] = mine[j * (NT * VEC / 32)] >> place32 & ALL;
                if (!MASK || allowed[j]) x[j] = sv[j * NT];
            }
        };
        const int last_whole = d1 - (BATCH - 1) * NT;  // a batch that starts before has no end in it
        const auto fetch_any = [&](int v) {
            if (!NEXT && v < last_whole)
                fetch(v, std::true_type());
            else
                fetch(v, std::false_type());
        };
        if (dense) fetch_any(d0);
        const bool simple = same && !p.in_place;
        const auto finish = [&](int v, int n_edit, auto whole) {
            uint4 *ov = reinterpret_cast<uint4 *>(out - shift) + v;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int u = v + j * NT, t = u * VEC - shift;
                if (!whole && u >= d1) break;
                if (MASK) cut(x[j], allowed[j], T());
                if (whole) {
                    ov[j * NT] = x[j];
                } else if (!p.in_place || (MASK && allowed[j] != ALL)) {
                    if (same) {
                        ov[j * NT] = x[j];
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) out[t + i] = reinterpret_cast<const T *>(&x[j])[i];
                    }
                }
                if (NEXT && (!MASK || allowed[j]) && top_of(x[j], T()) > top) {
                    const int w = t - t0;
                    const uint32_t skip = n_edit ? bits[w >> 5] >> (w & 31) : 0u;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float y = to_f(reinterpret_cast<const T *>(&x[j])[i]);
                        if (y > top && !(skip >> i & 1)) {
                            top = y;
                            at = t + i;
                        }
                    }
                }
            }
        };
        const auto dense_pass = [&](int n_edit) {
            for (int v = d0; v < d1; v += NT * BATCH) {
                if (v != d0) fetch_any(v);
                if (!NEXT && simple && v < last_whole)
                    finish(v, n_edit, std::true_type());
                else
                    finish(v, n_edit, std::false_type());
            }
            // the tokens of a row's first and last vector where those are not whole
            const int t = tid < VEC ? tid - shift : f1 * VEC - shift + tid - VEC;
            if (tid < 2 * VEC && inside(t) && (tid < VEC ? shift != 0 && t < VEC - shift : f1 >= f0)) {
                T y = in[t];
                const bool gone = masked(t);
                if (gone) from_f(-INFINITY, y);
                if (gone || !p.in_place) out[t] = y;
                if (NEXT && !(n_edit && (bits[(t - t0) >> 5] >> ((t - t0) & 31) & 1))) better(to_f(y), t);
            }
        };
        // Without a choice the pass needs nothing of the history, whose loads it then covers.
        if (!NEXT && dense) dense_pass(0);

        const unsigned below = (1u << lane) - 1;
        const uint32_t word0 = smem_u32(words);
        const auto listed = [&](int place, int w) {
            touched[place] = static_cast<uint16_t>(w);
            if (NEXT) atomicOr(&bits[w >> 5], 1u << (w & 31));
        };
        for (int i0 = warp * 32; i0 < r.nb; i0 += NT) {
            const int i = i0 + lane, t = i < r.nb ? btok[i] : -1;
            if (!inside(t)) continue;
            if (atomicMax(&words[t - t0], static_cast<uint32_t>(MAX_BIAS - i) << BIAS_AT))
                dups = 1;
            else
                listed(atomicAdd(&n_touched, 1), t - t0);
        }
        if (r.nb) __syncthreads();  // the counts go below the entries
        for (int i0 = warp * 32; i0 < n; i0 += NT * AHEAD) {
            if (i0 != warp * 32) tokens(i0);
            unsigned first[AHEAD];
            int many = 0;
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                first[k] = 0;
                if (i0 + k * NT >= n) continue;
                const bool here = inside(h[k]), early = i0 + k * NT + lane < from;
                const uint32_t before = counted(word0 + 4 * (h[k] - t0), here && early, here && !early);
                first[k] = __ballot_sync(0xFFFFFFFFu, before == 0);
                many += __popc(first[k]);
            }
            if (!many) continue;
            int place = 0;
            if (lane == 0) place = atomicAdd(&n_touched, many);
            place = __shfl_sync(0xFFFFFFFFu, place, 0);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (first[k] >> lane & 1) listed(place + __popc(first[k] & below), h[k] - t0);
                place += __popc(first[k]);
            }
        }
        __syncthreads();
        const int n_edit = n_touched;
        const float early = tid < n_edit ? to_f(in[t0 + touched[tid]]) : 0.0f;  // what the sparse pass needs first
        if (NEXT) {
            dense_pass(n_edit);
            __syncthreads();  // an edited logit replaces what the vectors wrote
        }

        for (int i = tid; i < n_edit; i += NT) {
            const int w = touched[i], t = t0 + w;
            const uint32_t word = words[w];
            words[w] = bits[w >> 5] = 0;
            if (masked(t)) continue;
            T y;
            from_f(edited(i == tid ? early : to_f(in[t]), word, r), y);
            out[t] = y;
            if (NEXT) better(to_f(y), t);
        }
    }
    __syncwarp();
    if (NEXT && p.cluster > 1) cluster_wait();
    if (NEXT) {
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
    if (NEXT && p.cluster > 1) cluster_sync_all();
    if (NEXT && tell) {
        unsigned long long key = row_best[0];
        for (int i = 1; i < p.cluster; ++i) key = max(key, row_best[i]);
        if (!key) atomicOr(p.status, ST_EDIT_NO_TOKEN);
        p.next[row] = key ? lin::argmax_key_index(key) : -1;
    }
}

typedef void (*Kernel)(Params);
template <typename T>
Kernel kernel(bool mask, bool next) {
    return mask ? (next ? k_logits_edit<T, true, true> : k_logits_edit<T, true, false>) : (next ? k_logits_edit<T, false, true> : k_logits_edit<T, false, false>);
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
    for (int i = 0; i < 4; ++i)
        for (const Kernel k : {kernel<__half>(i & 1, i & 2), kernel<float>(i & 1, i & 2)})
            if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (SEG + SEG / 16 + SEG / 2 + 2 * MAX_BIAS) * 4) != cudaSuccess) return GPT2_B200_ECUDA;
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
    // A row's CTAs: as many as run at once, and so many that a segment is all a CTA has, since each segment reads the history again.
    int c = 1;
    while (c < MAX_CLUSTER && vectors >= c * 128 && (static_cast<long long>(rows) * c * 2 <= 2ll * ctx->num_sms || vectors * vec > 1ll * c * SEG)) c *= 2;
    p.cluster = c;
    p.seg = static_cast<int>(std::min<long long>(SEG, ((vectors + c - 1) / c * vec + 127) / 128 * 128));  // what a warp looks at at once
    p.list = static_cast<int>(std::min<long long>(p.seg, ((e.history ? e.max_history : 0) + p.e.max_bias + 7ll) / 8 * 8));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * c, 1, 1);
    cfg.blockDim = dim3(NT, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.seg + p.seg / 16 + p.list / 2 + 2 * p.e.max_bias) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (c > 1 && next) {  // a row's CTAs meet only over its choice
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
    const Kernel k = type == GPT2_BEAM_HALF ? kernel<__half>(e.mask, next) : kernel<float>(e.mask, next);
    return cudaLaunchKernelEx(&cfg, k, p) == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
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
