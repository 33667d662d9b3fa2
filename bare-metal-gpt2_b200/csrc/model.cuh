// model.cuh — pieces of the GPT-2-124M decode step that its drivers share (internal): the sizes, the
// embedding and LayerNorm kernels, the launch helper and the check of a weight set.
#pragma once
#include "common.cuh"
#include "linear.cuh"
#include "ptx.cuh"

namespace b200 {
namespace model {

constexpr int E = 768, NL = 12, NH = 12, HD = 64, F = 3072, Q = 2304, V = 50257;
constexpr int LN_THREADS = 256;  // 3 elements per thread
constexpr float LN_EPS = 1e-5f;

// Block-wide sum of one float per thread (LN_THREADS threads).
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();  // red may still be read from a previous call
    if (lane == 0) red[warp] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < LN_THREADS / 32; ++w) s += red[w];
    return s;
}

// LayerNorm of one fp16 row held as 3 floats per thread; writes fp16 out.
// This thread's 3 elements of the LayerNorm gain and bias. They are weights, which no kernel of the
// step writes, so the LayerNorm kernels load them before their grid dependency wait: only the row
// itself is then read after it.
__device__ __forceinline__ void ln_params(const __half *g, const __half *bta, float (&gv)[3], float (&bv)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int e = threadIdx.x + i * LN_THREADS;
        gv[i] = __half2float(g[e]);
        bv[i] = __half2float(bta[e]);
    }
}

__device__ __forceinline__ void ln_row(const float (&xv)[3], __half *out, const float (&gv)[3],
                                       const float (&bv)[3], float *red) {
    const float mean = block_sum(xv[0] + xv[1] + xv[2], red) / E;
    float d2 = 0.0f;
#pragma unroll
    for (int i = 0; i < 3; ++i) d2 += (xv[i] - mean) * (xv[i] - mean);
    const float var = block_sum(d2, red) / E;
    const float inv = 1.0f / sqrtf(var + LN_EPS);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int e = threadIdx.x + i * LN_THREADS;
        out[e] = __float2half_rn((xv[i] - mean) * inv * gv[i] + bv[i]);
    }
}

// x[b] = fp16(wte[tok[b]] + wpe[pos[b]]); ln[b] = LayerNorm(x[b]) with layer 0's ln_1.
static __global__ void __launch_bounds__(LN_THREADS) k_embed_ln(__half *x, __half *ln, const __half *wte,
                                                         const __half *wpe, const __half *g,
                                                         const __half *bta, const int *tok,
                                                         const int *pos, int maxT, unsigned *status) {
    __shared__ float red[LN_THREADS / 32];
    float gv[3], bv[3];
    ln_params(g, bta, gv, bv);
    grid_dependency_wait();
    grid_launch_dependents();
    const int b = blockIdx.x;
    int t = tok[b], p = pos[b];
    if (t < 0 || t >= V || p < 0 || p >= maxT) {
        if (threadIdx.x == 0) atomicOr(status, ST_MODEL_BAD_TOKEN);
        t = min(max(t, 0), V - 1);
        p = min(max(p, 0), maxT - 1);
    }
    float xv[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int e = threadIdx.x + i * LN_THREADS;
        const __half h = __float2half_rn(__half2float(wte[static_cast<long long>(t) * E + e]) +
                                         __half2float(wpe[static_cast<long long>(p) * E + e]));
        x[static_cast<long long>(b) * E + e] = h;
        xv[i] = __half2float(h);
    }
    ln_row(xv, ln + static_cast<long long>(b) * E, gv, bv, red);
}

static __global__ void __launch_bounds__(LN_THREADS) k_layernorm(__half *ln, const __half *x,
                                                          const __half *g, const __half *bta) {
    __shared__ float red[LN_THREADS / 32];
    float gv[3], bv[3];
    ln_params(g, bta, gv, bv);
    grid_dependency_wait();
    grid_launch_dependents();
    const int b = blockIdx.x;
    float xv[3];
#pragma unroll
    for (int i = 0; i < 3; ++i)
        xv[i] = __half2float(x[static_cast<long long>(b) * E + threadIdx.x + i * LN_THREADS]);
    ln_row(xv, ln + static_cast<long long>(b) * E, gv, bv, red);
}

// Kernel launch, optionally as a programmatic dependent of the previous kernel in the stream (the
// kernels above all wait for their predecessor before touching memory it writes).
template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), int grid, int block, cudaStream_t st, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...) == cudaSuccess
               ? GPT2_B200_OK
               : GPT2_B200_ECUDA;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// linear: the four matmul weights of each layer are needed too (a batch over 4-bit weights has others).
inline bool weights_ok(const GPT2WeightsGPU *w, bool linear = true) {
    if (!w || !w->wte || !w->wpe || !w->lnf_g || !w->lnf_b || !aligned16(w->wte)) return false;
    for (int L = 0; L < NL; ++L) {
        const GPT2LayerGPU &l = w->layers[L];
        if (!l.ln1_g || !l.ln1_b || !l.qkv_b || !l.attn_proj_b || !l.ln2_g || !l.ln2_b || !l.fc_b || !l.proj_b) return false;
        if (!linear) continue;
        if (!l.qkv_w || !l.attn_proj_w || !l.fc_w || !l.proj_w) return false;
        if (!aligned16(l.qkv_w) || !aligned16(l.attn_proj_w) || !aligned16(l.fc_w) ||
            !aligned16(l.proj_w))
            return false;
    }
    return true;
}

}  // namespace model
}  // namespace b200
