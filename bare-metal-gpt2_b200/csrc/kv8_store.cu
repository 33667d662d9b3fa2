// kv8_store.cu — writing fp16 K/V rows into the paged 8-bit cache, and reading them back.
//
// Per unit = (block of positions, layer, K|V, head): s = max(s_old, amax / qmax), codes
// round(x * (1/s)); where an append makes s grow, the block's older codes become
// round(code * (s_old/s)). All in fp32 with IEEE division and multiplication, so the codes are a
// function of the inputs alone. Bound by HBM: 2 bytes in, 1 byte out per element (load: 1 in, 2 out).
//
// Store: a unit's new rows are read once, as 16-byte vectors that stay in registers (at most 8 per lane) from the
// maximum to the codes. A prompt's unit has a warp, or 2, 4 or 8 of them for blocks of over 2048 elements; a one-token
// append's unit, one row, has D / 8 lanes. An int8 code is rounded by adding 1.5 * 2^23 (the sum's low byte is
// the code, ties to even), which costs no conversion instruction.
// Load: a warp reads a head's 16 positions, four 8-byte vectors per lane in flight.
//
// Measured (8 sequences of 512 to 1023 positions x 12 layers x 12 heads x 64, int8): store 67 us, 5.1 TB/s of its 339 MB; load
// 72 us, 5.8 TB/s. One position of 64 sequences in 12 layers: 3.4 us.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace b200 {
namespace kv8 {

constexpr int NT = 256;
constexpr int VPL = 8;  // vectors per lane at most

// Eight halves: their largest magnitude (NaN or infinite if one of them is).
__device__ __forceinline__ float vec_amax(const uint4 &w) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&w);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    const __half x = __hmax_nan(__low2half(m), __high2half(m));
    return __half2float(x);
}
// NaN to 0, infinities to the largest fp16.
__device__ __forceinline__ void make_finite(uint4 &w) {
    __half *h = reinterpret_cast<__half *>(&w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = __half2float(h[j]);
        if (!(fabsf(x) <= 65504.0f)) h[j] = __float2half_rn(x != x ? 0.0f : copysignf(65504.0f, x));
    }
}
template <int KIND>
__device__ __forceinline__ uint2 encode8(const uint4 &w, float inv) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&w);
    uint32_t o[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 a = __half22float2(h[2 * k]), b = __half22float2(h[2 * k + 1]);
        if (KIND == GPT2_KV8_INT8) {  // |x * inv| <= 127 (1 + 2^-22): the rounded code never passes 127
            const uint32_t q0 = __float_as_uint(__fadd_rn(__fmul_rn(a.x, inv), 12582912.0f));
            const uint32_t q1 = __float_as_uint(__fadd_rn(__fmul_rn(a.y, inv), 12582912.0f));
            const uint32_t q2 = __float_as_uint(__fadd_rn(__fmul_rn(b.x, inv), 12582912.0f));
            const uint32_t q3 = __float_as_uint(__fadd_rn(__fmul_rn(b.y, inv), 12582912.0f));
            o[k] = __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
        } else {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a.x * inv, a.y * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(b.x * inv, b.y * inv), __NV_SATFINITE, __NV_E4M3);
            o[k] = lo | (hi << 16);
        }
    }
    return make_uint2(o[0], o[1]);
}
__device__ __forceinline__ uint4 ldg_stream(const __half *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// LPU lanes per unit (8 or 16: one row; 32 and up: a block), NV vectors per lane.
template <int KIND, int LPU, int NV>
__global__ void __launch_bounds__(NT)
    k_kv8_store(const View c, int L0, int units, const __half *k, const __half *v, long long layer_stride,
                long long row_stride, long long tok_stride, const int *d_count, int T, int spans) {
    constexpr int UPC = NT / LPU;  // units per CTA
    __shared__ float red[NT / 32];
    const int lane = threadIdx.x % LPU;
    const int r = blockIdx.x / spans, span = blockIdx.x - r * spans;
    const int unit = blockIdx.y * UPC + threadIdx.x / LPU;  // (layer, K|V, head)
    const bool ok_unit = unit < units;
    const int h = unit % c.nHead, lw = unit / c.nHead, which = lw & 1, l = lw >> 1;
    const int pos = c.len[r];
    const int n = d_count ? min(d_count[r], T) : T;
    const int cap = c.maxPages << c.page_shift;
    if (n < 0 || pos < 0 || pos > cap - n) {
        if (span == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        return;
    }
    const int b0 = ((pos >> c.block_shift) + span) << c.block_shift;  // first position of the block
    if (n == 0 || b0 >= pos + n) return;
    const int p = c.table[static_cast<long long>(r) * c.maxPages + (b0 >> c.page_shift)];
    if (p < 0 || p >= c.nPages) {
        if (blockIdx.y == 0 && threadIdx.x == 0) atomicOr(c.status, ST_KV8_BAD_PAGE);
        return;
    }
    const int lo = max(b0, pos), hi = min(b0 + c.block, pos + n);  // new positions
    const int vecs = c.D >> 3, vshift = c.D == 64 ? 3 : 4;         // 8-element vectors per position
    const int mine = ok_unit ? (hi - lo) * vecs : 0;
    const __half *src = (which ? v : k) + l * layer_stride + r * row_stride + (lo - pos) * tok_stride + static_cast<long long>(h) * c.D;
    const unsigned run = (static_cast<unsigned>(p) * c.nLayer + L0 + l) * 2 * c.nHead + which * c.nHead + h;
    const int in_page = b0 & (c.page - 1);
    float *sp = c.scale + (run << (c.page_shift - c.block_shift)) + (in_page >> c.block_shift);
    uint8_t *codes = c.data + ((static_cast<size_t>(run) << c.page_shift) + in_page) * c.D;
    const float s_old = ok_unit && pos > b0 ? *sp : 0.0f;
    uint4 x[NV];
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = lane + j * LPU;
        x[j] = i < mine ? ldg_stream(src + (i >> vshift) * tok_stride + ((i & (vecs - 1)) << 3)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        float a = vec_amax(x[j]);
        if (!(a <= 65504.0f)) {
            bad = true;
            make_finite(x[j]);
            a = vec_amax(x[j]);
        }
        amax = fmaxf(amax, a);
    }
#pragma unroll
    for (int o = (LPU < 32 ? LPU : 32) / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if (LPU > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
        __syncthreads();
        const int w0 = threadIdx.x / LPU * (LPU / 32);
#pragma unroll
        for (int w = 0; w < LPU / 32; ++w) amax = fmaxf(amax, red[w0 + w]);
    }
    const float s = fmaxf(s_old, amax / qmax<KIND>());
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    if (ok_unit && pos > b0 && s > s_old) {
        const float ratio = s_old / s;
        for (int i = lane; i < (pos - b0) * vecs; i += LPU) {
            uint2 w = reinterpret_cast<uint2 *>(codes)[i];
            uint8_t *q = reinterpret_cast<uint8_t *>(&w);
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = encode<KIND>(decode<KIND>(q[j]) * ratio);
            reinterpret_cast<uint2 *>(codes)[i] = w;
        }
    }
    uint2 *dst = reinterpret_cast<uint2 *>(codes + (lo - b0) * c.D);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = lane + j * LPU;
        if (i < mine) dst[i] = encode8<KIND>(x[j], inv);
    }
    __syncwarp();  // every lane of the unit has read *sp (the warps of a larger unit met at the barrier above)
    if (ok_unit && lane == 0 && (pos <= b0 || s > s_old)) *sp = s;
    if (bad) atomicOr(c.status, ST_KV8_NONFINITE);
}

// A warp per (row, 16-position granule, layer, K|V) and head, heads in turn.
template <int KIND, int D>
__global__ void __launch_bounds__(128)
    k_kv8_load(const View c, int L0, __half *k, __half *v, long long layer_stride, long long row_stride,
               long long tok_stride, const int *d_first, int T, const int *d_count, int count) {
    constexpr int VPR = D / 8, RPW = 32 / VPR, NL = 16 / RPW;  // vectors per row, rows per warp load, loads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.y, which = blockIdx.z & 1, l = blockIdx.z >> 1;
    const long long first = d_first ? d_first[r] : 0;
    const long long n = min(static_cast<long long>(c.len[r]) + (d_count ? d_count[r] : count),
                            static_cast<long long>(c.maxPages) << c.page_shift);
    const long long g0 = ((first >> 4) + blockIdx.x) << 4;  // the granule's first position (>> rounds down, also below 0)
    if (g0 >= first + T) return;
    bool ok = g0 >= 0 && g0 < n;
    int p = 0;
    if (ok) {
        p = c.table[static_cast<long long>(r) * c.maxPages + (g0 >> c.page_shift)];
        if (p < 0 || p >= c.nPages) {
            if (threadIdx.x == 0 && blockIdx.z == 0) atomicOr(c.status, ST_KV8_BAD_PAGE);
            ok = false;
        }
    }
    const int in_page = static_cast<int>(g0) & (c.page - 1);
    const unsigned run0 = (static_cast<unsigned>(p) * c.nLayer + L0 + l) * 2 * c.nHead + which * c.nHead;
    __half *out = (which ? v : k) + l * layer_stride + r * row_stride + (lane % VPR) * 8;
    for (int h = warp; h < c.nHead; h += 4) {
        const unsigned run = run0 + h;
        uint2 w[NL];
        float s = 0.0f;
        const uint8_t *src = c.data + ((static_cast<size_t>(run) << c.page_shift) + in_page + lane / VPR) * D + (lane % VPR) * 8;
        if (ok) {
            s = c.scale[(run << (c.page_shift - c.block_shift)) + (in_page >> c.block_shift)];
#pragma unroll
            for (int j = 0; j < NL; ++j) w[j] = __ldg(reinterpret_cast<const uint2 *>(src + j * RPW * D));
        }
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const long long at = g0 + j * RPW + lane / VPR;
            if (at < first || at >= first + T) continue;
            uint4 o = make_uint4(0, 0, 0, 0);
            if (ok && at < n) {
                const uint8_t *q = reinterpret_cast<const uint8_t *>(&w[j]);
                __half2 *y = reinterpret_cast<__half2 *>(&o);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = __floats2half2_rn(decode<KIND>(q[2 * i]) * s, decode<KIND>(q[2 * i + 1]) * s);
            }
            *reinterpret_cast<uint4 *>(out + (at - first) * tok_stride + h * D) = o;
        }
    }
}

static int check_rows(const GPT2KV8Cache *kv, int L0, int nL, const void *k, const void *v, long long ls,
                      long long rs, long long ts, int T) {
    if (check(kv) != GPT2_B200_OK || L0 < 0 || nL < 1 || L0 > kv->nLayer - nL || T < 0) return GPT2_B200_EINVAL;
    if (T == 0) return GPT2_B200_OK;
    if (!aligned(k) || !aligned(v) || (ls & 7) || (rs & 7) || (ts & 7) || nL > 32767) return GPT2_B200_EINVAL;
    return GPT2_B200_OK;
}

}  // namespace kv8
}  // namespace b200

using namespace b200;

extern "C" int gpt2_kv8_store_b200(const GPT2KV8Cache *kv, int L0, int nL, const gpt2_half *k,
                                   const gpt2_half *v, long long layer_stride, long long row_stride,
                                   long long tok_stride, const int *d_count, int T, cudaStream_t stream) {
    const int rc = kv8::check_rows(kv, L0, nL, k, v, layer_stride, row_stride, tok_stride, T);
    if (rc != GPT2_B200_OK || T == 0) return rc;
    if (T > kv->maxPages * kv->page) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    // Blocks that T positions at any offset can touch.
    const long long spans = (T + kv->block - 2) / kv->block + 1;
    const long long units = 2ll * nL * kv->nHead;
    const int vecs = kv->headDim / 8;
    // Lanes per unit: one row's vectors for one token; else a warp, or as many as keep a lane at VPL vectors.
    const int lpu = T == 1 ? vecs : std::max(32, kv->block * vecs / kv8::VPL), upc = kv8::NT / lpu;
    if (spans * kv->nRow > 0x7FFFFFFFll || units > 65535ll * upc) return GPT2_B200_EINVAL;
    const dim3 grid(static_cast<unsigned>(spans * kv->nRow), static_cast<unsigned>((units + upc - 1) / upc));
    auto go = [&](auto kern) {
        kern<<<grid, kv8::NT, 0, stream>>>(kv8::view(kv, ctx->status), L0, static_cast<int>(units), k, v, layer_stride, row_stride,
                                           tok_stride, d_count, T, static_cast<int>(spans));
        return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
    };
    const int nv = T == 1 ? 1 : kv->block * vecs / lpu;
    auto by_shape = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        if (lpu == 8) return go(kv8::k_kv8_store<KIND, 8, 1>);
        if (lpu == 16) return go(kv8::k_kv8_store<KIND, 16, 1>);
        if (lpu == 32 && nv == 4) return go(kv8::k_kv8_store<KIND, 32, 4>);
        if (lpu == 32) return go(kv8::k_kv8_store<KIND, 32, 8>);
        if (lpu == 64) return go(kv8::k_kv8_store<KIND, 64, 8>);
        if (lpu == 128) return go(kv8::k_kv8_store<KIND, 128, 8>);
        return go(kv8::k_kv8_store<KIND, 256, 8>);
    };
    return kv->kind == GPT2_KV8_INT8 ? by_shape(std::integral_constant<int, GPT2_KV8_INT8>())
                                     : by_shape(std::integral_constant<int, GPT2_KV8_E4M3>());
}

extern "C" int gpt2_kv8_load_b200(const GPT2KV8Cache *kv, int L0, int nL, gpt2_half *k, gpt2_half *v,
                                  long long layer_stride, long long row_stride, long long tok_stride,
                                  const int *d_first, int T, const int *d_count, int count, cudaStream_t stream) {
    const int rc = kv8::check_rows(kv, L0, nL, k, v, layer_stride, row_stride, tok_stride, T);
    if (rc != GPT2_B200_OK || T == 0) return rc;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    if (kv->nRow > 65535 || nL > 32767) return GPT2_B200_EINVAL;
    const dim3 grid((static_cast<unsigned>(T) + 14) / 16 + 1, kv->nRow, 2 * nL);  // granules that T positions at any offset touch
    auto go = [&](auto kern) {
        kern<<<grid, 128, 0, stream>>>(kv8::view(kv, ctx->status), L0, k, v, layer_stride, row_stride, tok_stride, d_first, T,
                                       d_count, count);
        return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
    };
    if (kv->kind == GPT2_KV8_INT8)
        return kv->headDim == 64 ? go(kv8::k_kv8_load<GPT2_KV8_INT8, 64>) : go(kv8::k_kv8_load<GPT2_KV8_INT8, 128>);
    return kv->headDim == 64 ? go(kv8::k_kv8_load<GPT2_KV8_E4M3, 64>) : go(kv8::k_kv8_load<GPT2_KV8_E4M3, 128>);
}
