// beam_select.cu — the next beams out of beams x vocabulary candidates.
//
// total(w, v) = score[w] + (x[w, v] - lse[w]), lse = max + log(sum exp(x - max)); a finished beam is the
// one candidate (w, eos) with its score. The W largest totals of an item, equal ones by the lower
// (w, v): candidates are compared as 64-bit keys, the total's bits made orderable above the inverted index.
//
// One CTA per item: a pass for the maxima, one for the sums, then W passes that each find the largest key
// below the one chosen before.
#include "kv8.cuh"
#include "linear.cuh"

namespace b200 {
namespace beam {

constexpr int MAX_W = 32;
constexpr int NT = 1024;

// NaN and +inf logits are no candidates (status bit): they count as -inf, like a masked token.
template <typename T>
__device__ __forceinline__ float logit(const T *p, bool &bad) {
    const float x = static_cast<float>(*p);
    if (x < INFINITY) return x;
    bad = true;
    return -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(NT)
    k_beam_select(int *token, int *parent, float *new_score, int *new_done, const T *logits, long long ld,
                  const float *score, const int *done, int W, int V, int eos, unsigned *status) {
    __shared__ float lse[MAX_W], sc[MAX_W];
    __shared__ int dn[MAX_W];
    __shared__ float red[32];
    __shared__ unsigned long long redk[32], best[MAX_W];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = logits + static_cast<long long>(b) * W * ld;
    bool bad = false;
    if (tid < W) {
        sc[tid] = score[b * W + tid];
        dn[tid] = done ? done[b * W + tid] : 0;
    }
    __syncthreads();
    for (int w = 0; w < W; ++w) {
        float top = -INFINITY;
        for (int v = tid; v < V; v += NT) top = fmaxf(top, logit(x + w * ld + v, bad));
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        __syncthreads();
        if (lane == 0) red[warp] = top;
        __syncthreads();
        top = red[lane];
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float sum = 0.0f;
        if (top > -INFINITY)
            for (int v = tid; v < V; v += NT) sum += expf(logit(x + w * ld + v, bad) - top);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        __syncthreads();
        if (lane == 0) red[warp] = sum;
        __syncthreads();
        sum = red[lane];
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (tid == 0) lse[w] = top + logf(sum);
    }
    if (bad) atomicOr(status, ST_BEAM_LOGIT);
    __syncthreads();
    unsigned long long prev = ~0ull;
    for (int k = 0; k < W; ++k) {
        unsigned long long key = 0;
        for (int w = 0; w < W; ++w) {
            if (!(sc[w] > -INFINITY)) continue;
            if (dn[w]) {
                const unsigned long long u = lin::argmax_key(sc[w], static_cast<unsigned>(w * V + max(eos, 0)));
                if (u < prev) key = max(key, u);
                continue;
            }
            for (int v = tid; v < V; v += NT) {
                const float l = logit(x + w * ld + v, bad);
                if (l == -INFINITY) continue;
                const unsigned long long u = lin::argmax_key(sc[w] + (l - lse[w]), static_cast<unsigned>(w * V + v));
                if (u < prev) key = max(key, u);
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long u = __shfl_xor_sync(0xFFFFFFFFu, key, o);
            key = max(key, u);
        }
        __syncthreads();
        if (lane == 0) redk[warp] = key;
        __syncthreads();
        key = redk[lane];
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long u = __shfl_xor_sync(0xFFFFFFFFu, key, o);
            key = max(key, u);
        }
        if (tid == 0) best[k] = key;
        prev = key;
        if (key == 0) {
            for (int j = k + 1 + tid; j < W; j += NT) best[j] = 0;
            break;
        }
    }
    __syncthreads();
    if (tid < W) {
        const unsigned long long key = best[tid];
        const int i = b * W + tid;
        if (key == 0) {  // fewer candidates than beams
            token[i] = max(eos, 0);
            parent[i] = i;
            new_score[i] = -INFINITY;
            if (new_done) new_done[i] = 1;
        } else {
            const unsigned idx = static_cast<unsigned>(lin::argmax_key_index(key));
            const int w = static_cast<int>(idx / V), v = static_cast<int>(idx - static_cast<unsigned>(w) * V);
            const unsigned o = static_cast<unsigned>(key >> 32);
            token[i] = v;
            parent[i] = b * W + w;
            new_score[i] = __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
            if (new_done) new_done[i] = dn[w] || v == eos;
        }
    }
}

}  // namespace beam
}  // namespace b200

using namespace b200;

extern "C" size_t gpt2_beam_work_bytes_b200(int B, int W) {
    if (B < 1 || W < 1 || W > beam::MAX_W) return 0;
    return 256;
}

extern "C" int gpt2_beam_select_b200(int *token, int *parent, float *new_score, int *new_done, const void *logits,
                                     int type, long long ld, const float *score, const int *done, int B, int W, int V,
                                     int eos, void *work, size_t work_bytes, cudaStream_t stream) {
    if (!token || !parent || !new_score || !logits || !score || !work || B < 0 || W < 1 || W > beam::MAX_W || V < 1 ||
        ld < V || eos < -1 || eos >= V || static_cast<long long>(W) * V > 0x7FFFFFFFll ||
        (type != GPT2_BEAM_HALF && type != GPT2_BEAM_FLOAT))
        return GPT2_B200_EINVAL;
    if (B == 0) return GPT2_B200_OK;
    if (work_bytes < gpt2_beam_work_bytes_b200(B, W)) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    if (type == GPT2_BEAM_HALF)
        beam::k_beam_select<<<B, beam::NT, 0, stream>>>(token, parent, new_score, new_done, static_cast<const __half *>(logits), ld,
                                                        score, done, W, V, eos, ctx->status);
    else
        beam::k_beam_select<<<B, beam::NT, 0, stream>>>(token, parent, new_score, new_done, static_cast<const float *>(logits), ld,
                                                        score, done, W, V, eos, ctx->status);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}
