// kv8_attend.cu — attention over the paged 8-bit cache.
//
// out = softmax(q K^T / sqrt(D)) V with K = code * scale per block: a block's scale is constant over
// its keys, so it multiplies the score of a key (K) and the probability (V) instead of every element.
// Online softmax in base 2: m, l and o are rescaled by 2^(m_old - m_new) per tile of keys.
//
// One warp per (row, query head, query): 32 keys a step, one key per lane for the scores, then D/32
// output dims per lane over the 32 probabilities.
#include "kv8.cuh"

namespace b200 {
namespace kv8 {

int attend_max_ctas() { return 2048; }

struct AttParams {
    const __half *q;
    __half *out;
    long long q_row, q_tok, o_row, o_tok;
    const int *d_first, *d_count;
    int L, Hq, Tq, count, max_len;
    float scale_log2;
};

template <int KIND, int D>
__global__ void __launch_bounds__(128) k_kv8_attend(const View c, const AttParams a) {
    const int lane = threadIdx.x & 31;
    const long long w = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (w >= static_cast<long long>(c.nRow) * a.Hq * a.Tq) return;
    const int t = static_cast<int>(w % a.Tq), hq = static_cast<int>(w / a.Tq % a.Hq), r = static_cast<int>(w / a.Tq / a.Hq);
    const int h = hq / (a.Hq / c.nHead);
    __shared__ float qs[4][D];
    float *q = qs[threadIdx.x >> 5];
    const __half *qp = a.q + r * a.q_row + t * a.q_tok + static_cast<long long>(hq) * D;
    for (int d = lane; d < D; d += 32) q[d] = __half2float(qp[d]) * a.scale_log2;
    __syncwarp();
    const int n = c.len[r] + (a.d_count ? a.d_count[r] : a.count);
    int first = a.d_first ? max(a.d_first[r], 0) : 0;
    int end = n - a.Tq + t + 1;  // keys [first, end)
    if (n < 0 || n > a.max_len) {
        if (lane == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        end = 0;
    }
    float m = -INFINITY, l = 0.0f, o[D / 32] = {};
    for (int j0 = first & ~31; j0 < end; j0 += 32) {
        const int j = j0 + lane;
        float s = -INFINITY, vs = 0.0f;
        long long vrow = 0;
        if (j >= first && j < end) {
            const int p = c.table[static_cast<long long>(r) * c.maxPages + (j >> c.page_shift)];
            if (p >= 0 && p < c.nPages) {
                const int ip = j & (c.page - 1), nb = c.page >> c.block_shift;
                const long long run = c.run(p, a.L, 0, h), vrun = run + c.nHead;
                const uint8_t *kp = c.data + ((run << c.page_shift) + ip) * D;
                float acc = 0.0f;
                for (int d = 0; d < D; d += 4) {
                    const unsigned x = *reinterpret_cast<const unsigned *>(kp + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc = fmaf(q[d + i], decode<KIND>((x >> (8 * i)) & 0xFFu), acc);
                }
                s = acc * c.scale[run * nb + (ip >> c.block_shift)];
                vs = c.scale[vrun * nb + (ip >> c.block_shift)];
                vrow = ((vrun << c.page_shift) + ip) * D;
            } else {
                atomicOr(c.status, ST_KV8_BAD_PAGE);
            }
        }
        float top = s;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        if (top == -INFINITY) continue;
        const float mn = fmaxf(m, top), f = exp2f(m - mn);
        const float p = exp2f(s - mn);
        m = mn;
        float sum = p;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
        l = l * f + sum;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= f;
        const float pv = p * vs;
        for (int jj = 0; jj < 32; ++jj) {
            const float pj = __shfl_sync(0xFFFFFFFFu, pv, jj);
            const long long row = __shfl_sync(0xFFFFFFFFu, vrow, jj);
            if (__shfl_sync(0xFFFFFFFFu, s, jj) == -INFINITY) continue;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] = fmaf(pj, decode<KIND>(c.data[row + lane + 32 * i]), o[i]);
        }
    }
    __half *op = a.out + r * a.o_row + t * a.o_tok + static_cast<long long>(hq) * D;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) op[lane + 32 * i] = __float2half_rn(o[i] * inv);
}

}  // namespace kv8
}  // namespace b200

using namespace b200;

extern "C" int gpt2_kv8_attend_b200(gpt2_half *out, long long out_row_stride, long long out_tok_stride,
                                    const gpt2_half *q, long long q_row_stride, long long q_tok_stride,
                                    const GPT2KV8Cache *kv, int L, int Hq, int Tq, const int *d_first,
                                    const int *d_count, int count, int max_len, cudaStream_t stream) {
    if (kv8::check(kv) != GPT2_B200_OK || L < 0 || L >= kv->nLayer || Hq < 1 || Hq % kv->nHead || Tq < 0 ||
        max_len < 0 || max_len > kv->maxPages * kv->page || count < 0)
        return GPT2_B200_EINVAL;
    if (Tq == 0) return GPT2_B200_OK;
    if (!kv8::aligned(out) || !kv8::aligned(q) || (out_row_stride & 7) || (out_tok_stride & 7) || (q_row_stride & 7) ||
        (q_tok_stride & 7) || kv->work_bytes < kv8::work_layout(kv, Hq, Tq).bytes)
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    kv8::AttParams a{q, out, q_row_stride, q_tok_stride, out_row_stride, out_tok_stride, d_first, d_count, L, Hq, Tq, count,
                     max_len ? max_len : kv->maxPages * kv->page,
                     1.4426950408889634f / sqrtf(static_cast<float>(kv->headDim))};
    const long long warps = static_cast<long long>(kv->nRow) * Hq * Tq;
    if ((warps + 3) / 4 > 0x7FFFFFFFll) return GPT2_B200_EINVAL;
    auto *kern = kv->kind == GPT2_KV8_INT8
                     ? (kv->headDim == 64 ? kv8::k_kv8_attend<GPT2_KV8_INT8, 64> : kv8::k_kv8_attend<GPT2_KV8_INT8, 128>)
                     : (kv->headDim == 64 ? kv8::k_kv8_attend<GPT2_KV8_E4M3, 64> : kv8::k_kv8_attend<GPT2_KV8_E4M3, 128>);
    kern<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, stream>>>(kv8::view(kv, ctx->status), a);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}
