// w4_pack.cu — fp16 weights to 4-bit codes with group scales and back (the format: w4.cuh).
//
// Both directions are one pass, bound by HBM: 2 bytes read and 0.5 + 2..4 / group written a weight, or the reverse. A CTA
// takes 32 rows x 256 k: a warp reads a row's 512 bytes in one instruction (8 elements a lane), 4 rows at once, finds the
// extremes of a group among its 4, 8 or 16 lanes, and writes one word of codes per lane. Scales are laid out by row,
// so they are collected in shared memory and leave as runs of 32 rows.
#include "w4.cuh"

namespace b200 {
namespace w4 {
namespace {

constexpr int ROWS = 32, COLS = 256, WARPS = 8, PER = ROWS / WARPS;

// x * inv to the nearest whole number in lo..hi, products rounded as they stand (no fused step: the codes do not depend on
// the compiler's choices).
__device__ __forceinline__ uint32_t code_of(float x, float inv, float lo, float hi) {
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(rintf(__fmul_rn(x, inv)), lo), hi)));
}

template <bool LEAST>
__global__ void __launch_bounds__(WARPS * 32)
    k_w4_quantize(uint32_t *codes, __half *scale, __half *least, const __half *W, long long ldw, int N, int K, int group, unsigned *status) {
    __shared__ __half sc[COLS / 32][ROWS], lo[COLS / 32][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_k = (K + COLS - 1) / COLS;
    const long long n0 = static_cast<long long>(blockIdx.x / tiles_k) * ROWS;
    const int k0 = blockIdx.x % tiles_k * COLS, k = k0 + lane * 8;
    const int span = group / 8;  // lanes of a group
    uint4 in[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long n = n0 + warp + i * WARPS;
        in[i] = make_uint4(0, 0, 0, 0);
        if (n < N && k < K) in[i] = __ldcs(reinterpret_cast<const uint4 *>(W + n * ldw + k));
    }
    bool odd = false;  // a value that is not finite
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int row = warp + i * WARPS;
        const long long n = n0 + row;
        float x[8];
        const __half2 *h = reinterpret_cast<const __half2 *>(&in[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(h[j]);
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!(fabsf(x[j]) <= 65504.0f)) {  // NaN counts as 0, infinities as the largest fp16
                odd = true;
                x[j] = x[j] != x[j] ? 0.0f : copysignf(65504.0f, x[j]);
            }
        }
        float top = LEAST ? x[0] : fabsf(x[0]), bottom = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            top = fmaxf(top, LEAST ? x[j] : fabsf(x[j]));
            bottom = fminf(bottom, x[j]);
        }
        for (int o = 1; o < span; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            if (LEAST) bottom = fminf(bottom, __shfl_xor_sync(0xFFFFFFFFu, bottom, o));
        }
        // The scale is rounded down, so that no code stands for a value outside the group's range (nor beyond fp16's); the
        // ends lose up to 15 * 2^-10 of a step by it, which a code's half step hides.
        const __half s = __float2half_rd(__fdiv_rn(LEAST ? __fsub_rn(top, bottom) : top, LEAST ? 15.0f : 7.0f));
        const float sf = __half2float(s), inv = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c = LEAST ? code_of(__fsub_rn(x[j], bottom), inv, 0.0f, 15.0f) : code_of(x[j], inv, -7.0f, 7.0f) + 8;
            word |= c << (j / 2 * 4 + j % 2 * 16);
        }
        if (n < N && k < K) codes[(n * K + k) >> 3] = word;
        if ((lane & (span - 1)) == 0) {
            sc[lane / span][row] = s;
            if (LEAST) lo[lane / span][row] = __float2half_rn(bottom);
        }
    }
    if (odd) atomicOr(status, ST_W4_NONFINITE);
    __syncthreads();
    const int groups = COLS / group;
    for (int i = threadIdx.x; i < groups * ROWS; i += WARPS * 32) {
        const int g = i / ROWS, row = i % ROWS;
        if (n0 + row >= N || k0 + g * group >= K) continue;
        const long long at = static_cast<long long>(k0 / group + g) * N + n0 + row;
        scale[at] = sc[g][row];
        if (LEAST) least[at] = lo[g][row];
    }
}

template <bool LEAST>
__global__ void __launch_bounds__(WARPS * 32)
    k_w4_dequantize(__half *W, long long ldw, const uint32_t *codes, const __half *scale, const __half *least, int N, int K, int group) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_k = (K + COLS - 1) / COLS;
    const long long n0 = static_cast<long long>(blockIdx.x / tiles_k) * ROWS;
    const int k = blockIdx.x % tiles_k * COLS + lane * 8;
    if (k >= K) return;
    uint32_t word[PER];
    __half s[PER], l[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long n = n0 + warp * PER + i;
        if (n >= N) break;
        const long long at = static_cast<long long>(k / group) * N + n;
        word[i] = __ldcs(codes + ((n * K + k) >> 3));
        s[i] = scale[at];
        if (LEAST) l[i] = least[at];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long n = n0 + warp * PER + i;
        if (n >= N) break;
        uint32_t v[4];
        values_of<LEAST, true>(word[i], scale_of<LEAST, true>(__half_as_ushort(s[i]), LEAST ? __half_as_ushort(l[i]) : 0), v);
        __stcs(reinterpret_cast<uint4 *>(W + n * ldw + k), make_uint4(v[0], v[1], v[2], v[3]));
    }
}

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Tiles of 32 x 256 in one grid dimension; 0 where there are too many.
unsigned tiles(const GPT2W4 *w) {
    const long long n = (static_cast<long long>(w->N) + ROWS - 1) / ROWS * ((w->K + COLS - 1) / COLS);
    return n <= 0x7FFFFFFFll ? static_cast<unsigned>(n) : 0u;
}

bool matrix_ok(const __half *W, long long ldw, const GPT2W4 *w) {
    return W && aligned(W, 16) && ldw >= w->K && (ldw & 7) == 0 && tiles(w) != 0;
}

}  // namespace

bool shape_ok(const GPT2W4 *w) {
    return w && (w->group == 32 || w->group == 64 || w->group == 128) && w->N >= 1 && w->K >= w->group && w->K % w->group == 0 && w->K <= (1 << 24);
}
bool weight_ok(const GPT2W4 *w) {
    return shape_ok(w) && w->codes && aligned(w->codes, 16) && w->scale && aligned(w->scale, 2) && aligned(w->least, 2);
}

}  // namespace w4
}  // namespace b200

using namespace b200;
using namespace b200::w4;

extern "C" {

int gpt2_w4_quantize_b200(const GPT2W4 *w, const gpt2_half *W, long long ldw, cudaStream_t stream) {
    if (!weight_ok(w) || !matrix_ok(W, ldw, w)) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    uint32_t *codes = static_cast<uint32_t *>(w->codes);
    if (w->least)
        k_w4_quantize<true><<<tiles(w), WARPS * 32, 0, stream>>>(codes, w->scale, w->least, W, ldw, w->N, w->K, w->group, ctx->status);
    else
        k_w4_quantize<false><<<tiles(w), WARPS * 32, 0, stream>>>(codes, w->scale, nullptr, W, ldw, w->N, w->K, w->group, ctx->status);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

int gpt2_w4_dequantize_b200(gpt2_half *W, long long ldw, const GPT2W4 *w, cudaStream_t stream) {
    if (!weight_ok(w) || !matrix_ok(W, ldw, w)) return GPT2_B200_EINVAL;
    if (!device_context()) return GPT2_B200_ECUDA;
    const uint32_t *codes = static_cast<const uint32_t *>(w->codes);
    if (w->least)
        k_w4_dequantize<true><<<tiles(w), WARPS * 32, 0, stream>>>(W, ldw, codes, w->scale, w->least, w->N, w->K, w->group);
    else
        k_w4_dequantize<false><<<tiles(w), WARPS * 32, 0, stream>>>(W, ldw, codes, w->scale, nullptr, w->N, w->K, w->group);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // extern "C"
