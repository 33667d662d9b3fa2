// w4_linear.cu — products with 4-bit weights: C[b, n] = e(sum_k x[b, k] * value(n, k) + bias[n]) for the B rows of a
// decoding step (the format and the values: w4.cuh).
#include <algorithm>

#include "w4.cuh"

namespace b200 {
namespace w4 {
namespace {

using lin::EPI_GELU;
using lin::EPI_HEAD;
using lin::EPI_QKV;
using lin::EPI_RESID;
using lin::EPI_STORE;

__device__ __forceinline__ float gelu_new(float v) {
    const float inner = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return 0.5f * v * (1.0f + tanhf(inner));
}

// One output of row b and feature n, both in range; acc holds the whole sum.
__device__ __forceinline__ __half put(const Dest &d, int b, int n, float acc) {
    if (d.bias) acc += __half2float(d.bias[n]);
    if (d.epi == EPI_GELU) acc = gelu_new(acc);
    if (d.epi == EPI_RESID) acc += __half2float(d.resid[b * d.ldr + n]);
    const __half h = __float2half_rn(acc);
    if (d.out) d.out[b * d.ldo + n] = h;
    if (d.epi == EPI_QKV && n >= d.E) {
        int m = n - d.E;
        const bool is_v = m >= d.E;
        if (is_v) m -= d.E;
        const int pos = d.d_pos[b];
        if (pos < 0 || pos >= d.maxT)
            atomicOr(d.status, ST_KV_BAD_POS);
        else
            (is_v ? d.v_dst[b] : d.k_dst[b])[(static_cast<long long>(m >> 6) * d.maxT + pos) * 64 + (m & 63)] = h;
    }
    return h;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- simple form: a warp per 16 features and 8 rows
// Lane (g, t) = (lane / 4, lane % 4) takes the 16 bytes of codes of features g and g + 8 at 32 neighbouring k; the matrix
// instructions sum over k in any order, so 4 of a lane's k serve as its share of each 16.
constexpr int CHUNK = 128;  // k per warp and step: 4 lanes x 32

template <bool LEAST>
__global__ void __launch_bounds__(32) k_w4_simple(const uint8_t *codes, const __half *scale, const __half *least, int K, int group, const __half *x, long long ldx,
                                                  const Dest d) {
    const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16, b0 = blockIdx.y * 8;
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    grid_dependency_wait();
    for (int k0 = 0; k0 < K; k0 += CHUNK) {
        const int k = k0 + 32 * t;
        uint4 q[2] = {};
        __half2 s[2] = {}, l[2] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = n0 + g + 8 * i;
            if (n < d.N && k < K) {
                q[i] = *reinterpret_cast<const uint4 *>(codes + (static_cast<long long>(n) * K + k) / 2);
                const long long at = static_cast<long long>(k / group) * d.N + n;
                s[i] = __half2half2(scale[at]);
                if (LEAST) l[i] = __half2half2(least[at]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 xv = make_uint4(0, 0, 0, 0);
            if (b0 + g < d.B && k < K) xv = *reinterpret_cast<const uint4 *>(x + (b0 + g) * ldx + k + 8 * j);
            uint32_t v[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) values_of<LEAST>((&q[i].x)[j], s[i], l[i], v[i]);
            const uint32_t a0[4] = {v[0][0], v[1][0], v[0][1], v[1][1]}, a1[4] = {v[0][2], v[1][2], v[0][3], v[1][3]};
            mma16816(c, a0, xv.x, xv.y);
            mma16816(c, a1, xv.z, xv.w);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + g + 8 * (i >> 1), b = b0 + 2 * t + (i & 1);
        const bool in = n < d.N && b < d.B;
        unsigned long long key = 0;
        if (in) {
            const float h = __half2float(put(d, b, n, c[i]));
            if (h == h) key = lin::argmax_key(h + 0.0f, static_cast<unsigned>(n));
        }
        if (d.epi == EPI_HEAD) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) key = max(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
            if (g == 0 && b < d.B) {
                unsigned long long *at = d.amax + static_cast<long long>(b) * d.keys + blockIdx.x;
                *at = i < 2 ? key : max(key, *at);
            }
        }
    }
}

}  // namespace

int keys_of(const GPT2W4 &w, int) { return (w.N + 15) / 16; }

int plan(Plan *pl, int epi, const GPT2W4 &w, const __half *x, long long ldx, int B, const __half *bias, __half *out, long long ldo) {
    if (!weight_ok(&w) || !x || (reinterpret_cast<uintptr_t>(x) & 15) || (ldx & 7) || ldx < w.K || B < 1 || B > lin::MAX_BPAD) return GPT2_B200_EINVAL;
    if (epi < EPI_STORE || epi > EPI_HEAD || (epi != EPI_HEAD && !out) || (out && ldo < w.N) ||
        ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1))
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    *pl = Plan{};
    pl->w = w;
    pl->x = x;
    pl->ldx = ldx;
    pl->d.epi = epi;
    pl->d.B = B;
    pl->d.N = w.N;
    pl->d.bias = bias;
    pl->d.out = out;
    pl->d.ldo = ldo;
    pl->d.keys = keys_of(w, B);
    pl->d.status = ctx->status;
    return GPT2_B200_OK;
}

int prepare(const Plan &) { return GPT2_B200_OK; }

int launch(const Plan &pl, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((pl.d.N + 15) / 16, (pl.d.B + 7) / 8, 1);
    cfg.blockDim = dim3(32, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pl.pdl ? 1 : 0;
    const uint8_t *codes = static_cast<const uint8_t *>(pl.w.codes);
    const auto go = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, codes, static_cast<const __half *>(pl.w.scale), static_cast<const __half *>(pl.w.least), pl.w.K, pl.w.group, pl.x, pl.ldx, pl.d); };
    return (pl.w.least ? go(k_w4_simple<true>) : go(k_w4_simple<false>)) == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace w4
}  // namespace b200

using namespace b200;

extern "C" int gpt2_w4_linear_b200(gpt2_half *C, long long ldc, const gpt2_half *A, long long lda, const GPT2W4 *w, const gpt2_half *bias, const gpt2_half *R,
                                   long long ldr, int B, int epi, cudaStream_t stream) {
    if (!w || !C || epi < GPT2_B200_LINEAR_STORE || epi > GPT2_B200_LINEAR_RESID || (epi == GPT2_B200_LINEAR_RESID && (!R || (reinterpret_cast<uintptr_t>(R) & 1) || ldr < w->N)))
        return GPT2_B200_EINVAL;
    w4::Plan pl;
    const int rc = w4::plan(&pl, epi == GPT2_B200_LINEAR_STORE ? lin::EPI_STORE : epi == GPT2_B200_LINEAR_GELU ? lin::EPI_GELU : lin::EPI_RESID, *w, A, lda, B, bias, C, ldc);
    if (rc != GPT2_B200_OK) return rc;
    pl.d.resid = R;
    pl.d.ldr = ldr;
    return w4::launch(pl, stream);
}
