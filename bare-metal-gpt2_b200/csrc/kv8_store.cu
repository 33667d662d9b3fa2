// kv8_store.cu — writing fp16 K/V rows into the paged 8-bit cache, and reading them back.
//
// Per unit = (block of positions, layer, K|V, head): s = max(s_old, amax / qmax), codes
// round(x * (1/s)); where an append makes s grow, the block's older codes become
// round(code * (s_old/s)). All in fp32 with IEEE division and multiplication, so the codes are a
// function of the inputs alone. Bound by HBM: 2 bytes in, 1 byte out per element.
//
// One warp per unit: a first pass over the block's new rows for amax (the rows come back from L1 for
// the second), 16-byte loads, 8-byte code stores.
#include "kv8.cuh"

namespace b200 {
namespace kv8 {

constexpr int WARPS = 4;

__device__ __forceinline__ float finite_or(float x, bool &bad) {
    if (fabsf(x) <= 65504.0f) return x;
    bad = true;
    return x != x ? 0.0f : copysignf(65504.0f, x);
}

template <int KIND>
__global__ void __launch_bounds__(32 * WARPS)
    k_kv8_store(const View c, int L0, int nL, const __half *k, const __half *v, long long layer_stride,
                long long row_stride, long long tok_stride, const int *d_count, int T, int spans) {
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.x / spans, span = blockIdx.x - r * spans;
    const int unit = blockIdx.y * WARPS + (threadIdx.x >> 5);  // (layer, K|V, head)
    if (unit >= nL * 2 * c.nHead) return;
    const int h = unit % c.nHead, which = (unit / c.nHead) & 1, l = unit / (2 * c.nHead);
    const int pos = c.len[r];
    const int n = d_count ? min(d_count[r], T) : T;
    const int cap = c.maxPages << c.page_shift;
    if (n < 0 || pos < 0 || pos > cap - n) {
        if (span == 0 && unit == 0 && lane == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        return;
    }
    const int b0 = ((pos >> c.block_shift) + span) << c.block_shift;  // first position of the block
    if (n == 0 || b0 >= pos + n) return;
    const int p = c.table[static_cast<long long>(r) * c.maxPages + (b0 >> c.page_shift)];
    if (p < 0 || p >= c.nPages) {
        if (unit == 0 && lane == 0) atomicOr(c.status, ST_KV8_BAD_PAGE);
        return;
    }
    const int lo = max(b0, pos), hi = min(b0 + c.block, pos + n);  // new positions
    const __half *src = (which ? v : k) + l * layer_stride + r * row_stride + static_cast<long long>(h) * c.D;
    const int vecs = c.D >> 3;  // 8-element vectors per position
    bool bad = false;
    float amax = 0.0f;
    for (int i = lane; i < (hi - lo) * vecs; i += 32) {
        const int t = i / vecs, d = (i - t * vecs) << 3;
        const uint4 w = *reinterpret_cast<const uint4 *>(src + (lo - pos + t) * tok_stride + d);
        const __half2 *h2 = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(h2[j]);
            amax = fmaxf(amax, fmaxf(fabsf(finite_or(f.x, bad)), fabsf(finite_or(f.y, bad))));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const long long run = c.run(p, L0 + l, which, h);
    const int in_page = b0 & (c.page - 1);
    float *sp = c.scale + run * (c.page >> c.block_shift) + (in_page >> c.block_shift);
    uint8_t *codes = c.data + (run << c.page_shift) * c.D + static_cast<long long>(in_page) * c.D;
    const float s_old = pos > b0 ? *sp : 0.0f;
    const float s = fmaxf(s_old, amax / qmax<KIND>());
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    if (pos > b0 && s > s_old) {
        const float ratio = s_old / s;
        for (int i = lane; i < (pos - b0) * vecs; i += 32) {
            uint2 w = reinterpret_cast<uint2 *>(codes)[i];
            uint8_t *q = reinterpret_cast<uint8_t *>(&w);
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = encode<KIND>(decode<KIND>(q[j]) * ratio);
            reinterpret_cast<uint2 *>(codes)[i] = w;
        }
    }
    for (int i = lane; i < (hi - lo) * vecs; i += 32) {
        const int t = i / vecs, d = (i - t * vecs) << 3;
        const uint4 w = *reinterpret_cast<const uint4 *>(src + (lo - pos + t) * tok_stride + d);
        const __half *x = reinterpret_cast<const __half *>(&w);
        uint2 o;
        uint8_t *q = reinterpret_cast<uint8_t *>(&o);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = encode<KIND>(finite_or(__half2float(x[j]), bad) * inv);
        *reinterpret_cast<uint2 *>(codes + (lo - b0 + t) * c.D + d) = o;
    }
    __syncwarp();
    if (lane == 0) *sp = s;
    if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(c.status, ST_KV8_NONFINITE);
}

// One thread per 8 elements of a row read back.
template <int KIND>
__global__ void __launch_bounds__(256)
    k_kv8_load(const View c, int L0, int nL, __half *k, __half *v, long long layer_stride,
               long long row_stride, long long tok_stride, const int *d_first, int T, const int *d_count,
               int count) {
    const int vecs = c.D >> 3;
    const int per_tok = c.nHead * vecs;
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= static_cast<long long>(T) * per_tok) return;
    const int t = static_cast<int>(i / per_tok), e = static_cast<int>(i - static_cast<long long>(t) * per_tok);
    const int r = blockIdx.y, which = blockIdx.z & 1, l = blockIdx.z >> 1;
    const int h = e / vecs, d = (e - h * vecs) << 3;
    const long long at = static_cast<long long>(d_first ? d_first[r] : 0) + t;
    const long long n = static_cast<long long>(c.len[r]) + (d_count ? d_count[r] : count);
    uint4 o = make_uint4(0, 0, 0, 0);
    const long long cap = static_cast<long long>(c.maxPages) << c.page_shift;
    if (at >= 0 && at < n && at < cap) {
        const int p = c.table[static_cast<long long>(r) * c.maxPages + (at >> c.page_shift)];
        if (p >= 0 && p < c.nPages) {
            const long long run = c.run(p, L0 + l, which, h);
            const int in_page = static_cast<int>(at) & (c.page - 1);
            const float s = c.scale[run * (c.page >> c.block_shift) + (in_page >> c.block_shift)];
            const uint2 w = *reinterpret_cast<const uint2 *>(c.data + ((run << c.page_shift) + in_page) * c.D + d);
            const uint8_t *q = reinterpret_cast<const uint8_t *>(&w);
            __half *x = reinterpret_cast<__half *>(&o);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __float2half_rn(decode<KIND>(q[j]) * s);
        } else if (e == 0 && blockIdx.z == 0) {
            atomicOr(c.status, ST_KV8_BAD_PAGE);
        }
    }
    *reinterpret_cast<uint4 *>((which ? v : k) + l * layer_stride + r * row_stride + t * tok_stride + (e << 3)) = o;
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
    if (spans * kv->nRow > 0x7FFFFFFFll || units > 65535ll * kv8::WARPS) return GPT2_B200_EINVAL;
    const dim3 grid(static_cast<unsigned>(spans * kv->nRow), static_cast<unsigned>((units + kv8::WARPS - 1) / kv8::WARPS));
    auto *kern = kv->kind == GPT2_KV8_INT8 ? kv8::k_kv8_store<GPT2_KV8_INT8> : kv8::k_kv8_store<GPT2_KV8_E4M3>;
    kern<<<grid, 32 * kv8::WARPS, 0, stream>>>(kv8::view(kv, ctx->status), L0, nL, k, v, layer_stride, row_stride,
                                               tok_stride, d_count, T, static_cast<int>(spans));
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

extern "C" int gpt2_kv8_load_b200(const GPT2KV8Cache *kv, int L0, int nL, gpt2_half *k, gpt2_half *v,
                                  long long layer_stride, long long row_stride, long long tok_stride,
                                  const int *d_first, int T, const int *d_count, int count, cudaStream_t stream) {
    const int rc = kv8::check_rows(kv, L0, nL, k, v, layer_stride, row_stride, tok_stride, T);
    if (rc != GPT2_B200_OK || T == 0) return rc;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    const long long blocks = (static_cast<long long>(T) * kv->nHead * (kv->headDim / 8) + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return GPT2_B200_EINVAL;
    const dim3 grid(static_cast<unsigned>(blocks), kv->nRow, 2 * nL);
    auto *kern = kv->kind == GPT2_KV8_INT8 ? kv8::k_kv8_load<GPT2_KV8_INT8> : kv8::k_kv8_load<GPT2_KV8_E4M3>;
    kern<<<grid, 256, 0, stream>>>(kv8::view(kv, ctx->status), L0, nL, k, v, layer_stride, row_stride, tok_stride,
                                   d_first, T, d_count, count);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}
