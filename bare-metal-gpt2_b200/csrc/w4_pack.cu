// w4_pack.cu — fp16 weights to 4-bit codes with group scales and back (the format: w4.cuh).
//
// Both directions are one pass, bound by HBM: 2 bytes read and 0.5 + 2..4 / group written a weight, or the reverse. A CTA
// takes 32 rows x 256 k: a warp reads a row's 512 bytes in one instruction (8 elements a lane), 4 rows at once, finds the
// extremes of a group among its 4, 8 or 16 lanes, and writes one word of codes per lane. At HBM's rate a warp has about 28 cycles
// of an SM for its 256 weights, so instructions count: extremes are found in packed fp16 (exact), the divisions of 4 rows are
// done once, in different lanes, and a product becomes a whole number by adding 1.5 * 2^23 to it. Scales are laid out by row, so they are
// collected in shared memory and leave as runs of 32 rows. 8192 x 8192 with least, both ways: 68 us, 5.0 TB/s (floor 52); quantising issues at
// 85% of the slots.
#include "w4.cuh"

namespace b200 {
namespace w4 {
namespace {

constexpr int ROWS = 32, COLS = 256, WARPS = 8, PER = ROWS / WARPS;

__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ __half2 pair_of(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }

template <bool LEAST>
__global__ void __launch_bounds__(WARPS * 32)
    k_w4_quantize(uint32_t *codes, __half *scale, __half *least, const __half *W, long long ldw, int N, int K, int group, unsigned *status) {
    __shared__ __half sc[COLS / 32][ROWS], lo[COLS / 32][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_k = (K + COLS - 1) / COLS;
    const long long n0 = static_cast<long long>(blockIdx.x / tiles_k) * ROWS;
    const int k0 = blockIdx.x % tiles_k * COLS, k = k0 + lane * 8;
    const int span = group / 8;  // lanes of a group: 4 at least, one for each of the warp's rows
    uint4 in[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long n = n0 + warp + i * WARPS;
        in[i] = make_uint4(0, 0, 0, 0);
        if (n < N && k < K) in[i] = __ldcs(reinterpret_cast<const uint4 *>(W + n * ldw + k));
    }
    // A row's extremes as one register: (largest, -smallest), or the largest magnitude twice.
    __half2 ends[PER];
    bool odd = false;  // a value that is not finite
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        uint32_t *w = &in[i].x;
        const uint32_t some = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
        const uint32_t big = max(some & 0xFFFFu, some >> 16);
        if (big >= 0x7C00u) {  // NaN counts as 0, infinities as the largest fp16
            odd = true;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int half = 0; half < 32; half += 16) {
                    const uint32_t m = w[j] >> half & 0x7FFFu;
                    if (m > 0x7C00u) w[j] &= ~(0xFFFFu << half);
                    if (m == 0x7C00u) w[j] -= 1u << half;
                }
        }
        const __half2 a = pair_of(w[0]), b = pair_of(w[1]), c = pair_of(w[2]), d = pair_of(w[3]);
        if (LEAST) {
            const __half2 up = __hmax2(__hmax2(a, b), __hmax2(c, d)), down = __hmin2(__hmin2(a, b), __hmin2(c, d));
            ends[i] = __halves2half2(__hmax(__low2half(up), __high2half(up)), __hneg(__hmin(__low2half(down), __high2half(down))));
        } else {
            const __half2 up = __hmax2(__hmax2(__habs2(a), __habs2(b)), __hmax2(__habs2(c), __habs2(d)));
            ends[i] = __half2half2(__hmax(__low2half(up), __high2half(up)));
        }
    }
    for (int o = 1; o < span; o <<= 1)
#pragma unroll
        for (int i = 0; i < PER; ++i) ends[i] = __hmax2(ends[i], pair_of(__shfl_xor_sync(0xFFFFFFFFu, bits_of(ends[i]), o)));
    // Lane r of a group makes row r's scale. It is rounded down, so that no code stands for a value outside the group's range (nor beyond
    // fp16's); the ends lose up to 15 * 2^-10 of a step by it, which a code's half step hides.
    const int r = lane & 3;
    const __half2 own = r == 0 ? ends[0] : r == 1 ? ends[1] : r == 2 ? ends[2] : ends[3];
    const float top = __low2float(own), bottom = -__high2float(own);
    const __half s = __float2half_rd(__fdiv_rn(LEAST ? __fsub_rn(top, bottom) : top, LEAST ? 15.0f : 7.0f));
    const float sf = __half2float(s), inverse = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
    const int in_group = lane & (span - 1);
    if (in_group < PER) {
        sc[lane / span][warp + in_group * WARPS] = s;
        if (LEAST) lo[lane / span][warp + in_group * WARPS] = __float2half_rn(bottom);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long n = n0 + warp + i * WARPS;
        const float inv = __shfl_sync(0xFFFFFFFFu, inverse, (lane & ~(span - 1)) + i), low = -__high2float(ends[i]);
        const uint32_t *w = &in[i].x;
        // x * inv, as it is rounded to fp32, plus 1.5 * 2^23 (and 8) has the nearest whole number, ties to even, in its lowest bits; the bits
        // above are the same for all and are taken off at once. Clamped first: a subnormal scale is coarse.
        constexpr float magic = LEAST ? 12582912.0f : 12582920.0f;
        constexpr uint32_t base = 0x4B400000u;
        uint32_t word = 0u - (base + (base << 16) + (base << 4) + (base << 20) + (base << 8) + (base << 24) + (base << 12) + (base << 28));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(pair_of(w[j]));
            float y0 = __fmul_rn(LEAST ? __fsub_rn(f.x, low) : f.x, inv), y1 = __fmul_rn(LEAST ? __fsub_rn(f.y, low) : f.y, inv);
            y0 = fminf(y0, LEAST ? 15.0f : 7.0f);
            y1 = fminf(y1, LEAST ? 15.0f : 7.0f);
            if (!LEAST) {
                y0 = fmaxf(y0, -7.0f);
                y1 = fmaxf(y1, -7.0f);
            }
            word += __float_as_uint(__fadd_rn(y0, magic)) * (1u << (4 * j)) + __float_as_uint(__fadd_rn(y1, magic)) * (1u << (16 + 4 * j));
        }
        if (n < N && k < K) codes[(n * K + k) >> 3] = word;
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

// N: a feature's number, rounded up to a tile, is an int.
bool weight_ok(const GPT2W4 *w) {
    return w && (w->group == 32 || w->group == 64 || w->group == 128) && w->N >= 1 && w->N <= (1 << 30) && w->K >= w->group && w->K % w->group == 0 &&
           w->K <= (1 << 24) && w->codes && aligned(w->codes, 16) && w->scale && aligned(w->scale, 2) && aligned(w->least, 2);
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
