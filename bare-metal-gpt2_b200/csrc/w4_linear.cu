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
    // gelu_new, 0.5 v (1 + tanh u) = v / (1 + e^-2u), u = sqrt(2 / pi) (v + 0.044715 v^3): no cancellation where tanh nears -1
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return __fdividef(v, 1.0f + __expf(-2.0f * u));
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

// ---------------------------------------------------------------- tensor-core form
constexpr int BM = 128;                  // features of a tile: the MMA's M, one TMEM lane each
constexpr int KS = 128;                  // k of a stage
constexpr int CODE_BYTES = BM * KS / 2;  // 8 KB of codes
constexpr int CODE_RING = 8;             // stages of codes in flight (even: each warpgroup has slots of its own)
constexpr int X_ATOM = 64;               // k of a piece of x: one 128-byte swizzle row
constexpr int MAX_X_RING = 16;           // pieces of x in flight
constexpr int A_BUFS = 4;                // converted stages: TMEM columns of 64 each
constexpr int A_COLS = KS / 2;
constexpr int TC_THREADS = 512;
constexpr size_t TC_SMEM = 227 * 1024;  // the SM for itself: no other CTA's TMEM allocation meets this one's

struct TcParams {
    const __half *scale, *least;
    int K, group;
    int stages, cs, tiles;   // per tile; CTAs that share a tile's k; tiles
    int x_ring, bpad, nacc;  // pieces of x in flight; columns; accumulators
    Dest d;
    unsigned long long timeout_ns;
};

__device__ __forceinline__ float dsmem_ld_f32(uint32_t cluster_saddr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_saddr) : "memory");
    return v;
}

// Columns [c0, c1) of this warp's 32 features out of TMEM, through the epilogue. acc: the accumulator's first column.
__device__ __forceinline__ void epilogue(const Dest &d, uint32_t acc, int warp4, int lane, int n0, int tile, int c0, int c1) {
    const int n = n0 + warp4 * 32 + lane;
    const uint32_t row = acc + (static_cast<uint32_t>(warp4 * 32) << 16);
    for (int c = c0; c < c1; c += 16) {
        uint32_t r[16];
        tmem_ld16(row + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int b = c + j;
            if (b >= d.B) break;
            __half h = __float2half_rn(0.0f);
            if (n < d.N) h = put(d, b, n, __uint_as_float(r[j]));
            if (d.epi == EPI_HEAD) {
                const float v = __half2float(h) + 0.0f;
                const unsigned long long key = n < d.N && v == v ? lin::argmax_key(v, static_cast<unsigned>(n)) : 0ull;
                const unsigned hi = static_cast<unsigned>(key >> 32), mhi = __reduce_max_sync(0xFFFFFFFFu, hi);
                const unsigned mlo = __reduce_max_sync(0xFFFFFFFFu, hi == mhi ? static_cast<unsigned>(key) : 0u);
                if (lane == 0) d.amax[static_cast<long long>(b) * d.keys + tile * 4 + warp4] = static_cast<unsigned long long>(mhi) << 32 | mlo;
            }
        }
    }
}

// GS: groups per stage, 128 / group.
template <int GS, bool LEAST>
__global__ void __launch_bounds__(TC_THREADS, 1) k_w4_tc(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const TcParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t c_full[CODE_RING], c_empty[CODE_RING], x_full[MAX_X_RING], x_empty[MAX_X_RING], a_full[A_BUFS], a_empty[A_BUFS], acc_full[2],
        acc_empty[2], last_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int bad;  // a wait gave up: nothing more is written
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *const x_smem = smem + CODE_RING * CODE_BYTES;
    const int x_bytes = p.bpad * 2 * X_ATOM;
    const int rank = static_cast<int>(cluster_rank());
    const int first_tile = blockIdx.x / p.cs, tile_step = gridDim.x / p.cs;
    const int my_tiles = (p.tiles - first_tile + tile_step - 1) / tile_step;
    const int s0 = rank * p.stages / p.cs, ns = (rank + 1) * p.stages / p.cs - s0;  // this CTA's stages of each tile
    const int total = my_tiles * ns;

    if (tid == 0) {
        for (int i = 0; i < CODE_RING; ++i) {
            mbar_init(&c_full[i], 1);
            mbar_init(&c_empty[i], 4);
        }
        for (int i = 0; i < MAX_X_RING; ++i) {
            mbar_init(&x_full[i], 1);
            mbar_init(&x_empty[i], 1);
        }
        for (int i = 0; i < A_BUFS; ++i) {
            mbar_init(&a_full[i], 4);
            mbar_init(&a_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 4);
        }
        mbar_init(&last_full, 1);
        bad = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm_a = tmem_slot, tm_acc = tmem_slot + A_BUFS * A_COLS;
    grid_launch_dependents();

    const auto fail = [&] {
        if (lane == 0) {
            bad = 1;
            atomicOr(p.d.status, ST_LINEAR_TIMEOUT);
        }
    };
    if (warp == 0) {
        // Codes: they do not depend on the kernel before this one, so nothing waits for it.
        const bool leader = elect_one();
        int it = 0;
        for (; it < total; ++it) {
            const int slot = it % CODE_RING;
            const bool ok = it < CODE_RING || mbar_wait(&c_empty[slot], (it / CODE_RING - 1) & 1, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                fail();
                break;
            }
            if (leader) {
                mbar_arrive_expect_tx(&c_full[slot], CODE_BYTES);
                tma_load_2d(smem + slot * CODE_BYTES, &tm_w, &c_full[slot], (s0 + it % ns) * (KS / 2), (first_tile + it / ns * tile_step) * BM);
            }
            __syncwarp();
        }
        // every copy has landed before this CTA may end, whatever became of the others
        for (int i = max(0, it - CODE_RING); i < it; ++i) mbar_wait(&c_full[i % CODE_RING], (i / CODE_RING) & 1, p.timeout_ns);
    } else {
        grid_dependency_wait();
    }
    if (warp == 2) {
        const bool leader = elect_one();
        int at = 0;
        for (; at < 2 * total; ++at) {
            const int slot = at % p.x_ring;
            const bool ok = at < p.x_ring || mbar_wait(&x_empty[slot], (at / p.x_ring - 1) & 1, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                fail();
                break;
            }
            if (leader) {
                mbar_arrive_expect_tx(&x_full[slot], static_cast<uint32_t>(x_bytes));
                tma_load_2d(x_smem + slot * x_bytes, &tm_x, &x_full[slot], (s0 + at / 2 % ns) * KS + at % 2 * X_ATOM, 0);
            }
            __syncwarp();
        }
        for (int i = max(0, at - p.x_ring); i < at; ++i) mbar_wait(&x_full[i % p.x_ring], (i / p.x_ring) & 1, p.timeout_ns);
    }
    if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t idesc = idesc_f16_f32(BM, p.bpad, 0, 0);
        const uint64_t dx = sdesc_sw128(smem_u32(x_smem), 16, 1024);
        const uint32_t x_lo = static_cast<uint32_t>(dx), x_hi = static_cast<uint32_t>(dx >> 32);
        int it = 0;
        bool ok = true;
        for (int j = 0; j < my_tiles && ok; ++j) {
            const int acc = j % p.nacc;
            if (j >= p.nacc) ok = __all_sync(0xFFFFFFFFu, mbar_wait_spin(&acc_empty[acc], (j / p.nacc - 1) & 1, p.timeout_ns));
            for (int i = 0; i < ns && ok; ++i, ++it) {
                const int buf = it % A_BUFS;
                ok = mbar_wait_spin(&a_full[buf], (it / A_BUFS) & 1, p.timeout_ns);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = 2 * it + h, slot = at % p.x_ring;
                    ok = ok && mbar_wait_spin(&x_full[slot], (at / p.x_ring) & 1, p.timeout_ns);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
                        const uint32_t off = static_cast<uint32_t>(slot * x_bytes) >> 4;
#pragma unroll
                        for (int kk = 0; kk < X_ATOM / 16; ++kk)
                            umma_f16_ts_lohi(tm_acc + acc * p.bpad, tm_a + buf * A_COLS + h * (X_ATOM / 2) + kk * 8, x_lo + off + kk * 2, x_hi, idesc,
                                             i > 0 || h > 0 || kk > 0 ? 1u : 0u);
                        umma_commit(&x_empty[slot]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) {
                    umma_commit(&a_empty[buf]);
                    if (i == ns - 1) umma_commit(&acc_full[acc]);
                }
                __syncwarp();
            }
        }
        if (!ok) fail();
        __syncwarp();
        if (leader) umma_commit(&last_full);  // arrives when all that was issued is done
    } else if (warp >= 4 && warp < 12) {
        // Two warpgroups take every other stage: a thread converts the 128 codes of one feature, 64 TMEM columns.
        const int wg = (warp - 4) >> 2, warp4 = warp & 3, row = warp4 * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(warp4 * 32) << 16;
        const int groups = p.K / p.group;
        __half sc[2][GS], lo[2][GS];
        const auto scales = [&](int it, __half (&s)[GS], __half (&l)[GS]) {
            const int n = (first_tile + it / ns * tile_step) * BM + row;
            const int g0 = (s0 + it % ns) * GS;
#pragma unroll
            for (int q = 0; q < GS; ++q) {
                const bool in = it < total && n < p.d.N && g0 + q < groups;
                const long long at = static_cast<long long>(g0 + q) * p.d.N + n;
                s[q] = in ? p.scale[at] : __float2half_rn(0.0f);
                if (LEAST) l[q] = in ? p.least[at] : __float2half_rn(0.0f);
            }
        };
        scales(wg, sc[0], lo[0]);
        scales(wg + 2, sc[1], lo[1]);
        bool ok = true;
        for (int it0 = wg; it0 < total && ok; it0 += 4) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int it = it0 + 2 * u;
                if (it >= total || !ok) break;
                const int slot = it % CODE_RING, buf = it % A_BUFS;
                ok = mbar_wait(&c_full[slot], (it / CODE_RING) & 1, p.timeout_ns);
                if (it >= A_BUFS) ok = ok && mbar_wait(&a_empty[buf], (it / A_BUFS - 1) & 1, p.timeout_ns);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint8_t *st = smem + slot * CODE_BYTES + row * 64;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[32];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int chunk = h * 2 + q;  // 32 k, 16 bytes: the 64-byte swizzle's place
                        const uint4 w = *reinterpret_cast<const uint4 *>(st + ((chunk ^ (row >> 1 & 3)) << 4));
                        const __half2 s2 = __half2half2(sc[u][chunk * GS / 4]), l2 = LEAST ? __half2half2(lo[u][chunk * GS / 4]) : s2;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t four[4];
                            values_of<LEAST>((&w.x)[j], s2, l2, four);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[q * 16 + j * 4 + e] = four[e];
                        }
                    }
                    tmem_st32(tm_a + lanes + buf * A_COLS + h * 32, v);
                }
                scales(it + 4, sc[u], lo[u]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&c_empty[slot]);
                    mbar_arrive(&a_full[buf]);
                }
            }
        }
        if (!ok) fail();
    }
    __syncwarp();

    // The epilogue warps take each tile as it is done; at the last one, when nothing is left to convert, the others help.
    if (warp >= 4) {
        const int wg = (warp - 4) >> 2, warp4 = warp & 3;  // 2: the epilogue's own
        for (int j = wg == 2 ? 0 : my_tiles - 1; j < my_tiles; ++j) {
            const int acc = j % p.nacc, tile = first_tile + j * tile_step;
            const int cols = p.bpad / 16;
            const bool last = j == my_tiles - 1;
            const bool ok = last ? mbar_wait(&last_full, 0, p.timeout_ns) : mbar_wait(&acc_full[acc], (j / p.nacc) & 1, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) fail();
            __syncwarp();
            if (*reinterpret_cast<volatile int *>(&bad)) break;
            tc_fence_after();
            const int c0 = last ? wg * cols / 3 * 16 : 0, c1 = last ? (wg + 1) * cols / 3 * 16 : p.bpad;
            if (p.cs == 1) {
                epilogue(p.d, tm_acc + acc * p.bpad, warp4, lane, tile * BM, tile, c0, c1);
            } else {
                float *part = reinterpret_cast<float *>(smem);  // the ring has been read: [column][feature]
                const uint32_t row = tm_acc + acc * p.bpad + (static_cast<uint32_t>(warp4 * 32) << 16);
                for (int c = c0; c < c1; c += 16) {
                    uint32_t r[16];
                    tmem_ld16(row + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * BM + warp4 * 32 + lane] = __uint_as_float(r[i]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (!last && lane == 0) mbar_arrive(&acc_empty[acc]);
        }
    }
    __syncwarp();
    if (p.cs > 1) {
        // Each CTA of the cluster sums its share of the columns over the ranks, in their order.
        cluster_sync_all();
        const uint32_t part = smem_u32(smem) + (tid & (BM - 1)) * 4;
        const int n = first_tile * BM + (tid & (BM - 1));
        const int b1 = min(p.d.B, (rank + 1) * p.bpad / p.cs);
        for (int b = rank * p.bpad / p.cs + tid / BM; b < b1; b += TC_THREADS / BM) {
            float v[lin::MAX_CLUSTER];
#pragma unroll
            for (int q = 0; q < lin::MAX_CLUSTER; ++q)
                if (q < p.cs) v[q] = dsmem_ld_f32(dsmem_addr(part + b * BM * 4, static_cast<uint32_t>(q)));
            float sum = v[0];
#pragma unroll
            for (int q = 1; q < lin::MAX_CLUSTER; ++q)
                if (q < p.cs) sum += v[q];
            if (n < p.d.N && !*reinterpret_cast<volatile int *>(&bad)) put(p.d, b, n, sum);
        }
        cluster_sync_all();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_slot, 512);
}

}  // namespace

namespace {

constexpr int SIMPLE_MAX_B = 0;

typedef void (*TcKernel)(CUtensorMap, CUtensorMap, TcParams);
template <bool LEAST>
TcKernel tc_kernel(int group) {
    return group == 128 ? k_w4_tc<1, LEAST> : group == 64 ? k_w4_tc<2, LEAST> : k_w4_tc<4, LEAST>;
}
TcKernel tc_kernel(const GPT2W4 &w) { return w.least ? tc_kernel<true>(w.group) : tc_kernel<false>(w.group); }

bool encode(CUtensorMap *m, CUtensorMapDataType type, const void *ptr, long long inner, long long rows, long long row_bytes, int box_inner, int box_rows,
            CUtensorMapSwizzle swizzle) {
    const EncodeTiledFn fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
    return fn(m, type, 2, const_cast<void *>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many clusters of cs CTAs run at once (one CTA per SM), asked once per device.
int active_clusters(DeviceContext *ctx, int cs) {
    int &n = ctx->w4_clusters[cs];
    if (n) return n;
    RelaxedCapture relaxed;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(cs) * 64, 1, 1);
    cfg.blockDim = dim3(TC_THREADS, 1, 1);
    cfg.dynamicSmemBytes = TC_SMEM - 1024;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cs);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, k_w4_tc<1, false>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n = got;
}

int prepare_tc(DeviceContext *ctx) {
    if (ctx->w4_attr_done) return GPT2_B200_OK;
    RelaxedCapture relaxed;
    for (const TcKernel k : {k_w4_tc<1, false>, k_w4_tc<2, false>, k_w4_tc<4, false>, k_w4_tc<1, true>, k_w4_tc<2, true>, k_w4_tc<4, true>})
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(TC_SMEM - 1024)) != cudaSuccess) return GPT2_B200_ECUDA;
    ctx->w4_attr_done = true;
    return GPT2_B200_OK;
}

}  // namespace

int keys_of(const GPT2W4 &w, int B) { return B <= SIMPLE_MAX_B ? (w.N + 15) / 16 : (w.N + BM - 1) / BM * 4; }

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

namespace {

int launch_simple(const Plan &pl, cudaStream_t stream) {
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

int launch_tc(DeviceContext *ctx, const Plan &pl, cudaStream_t stream) {
    const int rc = prepare_tc(ctx);
    if (rc != GPT2_B200_OK) return rc;
    const GPT2W4 &w = pl.w;
    TcParams p = {};
    p.scale = w.scale;
    p.least = w.least;
    p.K = w.K;
    p.group = w.group;
    p.stages = (w.K + KS - 1) / KS;
    p.tiles = (w.N + BM - 1) / BM;
    p.bpad = (pl.d.B + 15) / 16 * 16;
    p.nacc = p.bpad <= 128 ? 2 : 1;
    p.d = pl.d;
    p.timeout_ns = wait_timeout_ns();
    p.x_ring = std::min<int>(MAX_X_RING, static_cast<int>((TC_SMEM - 3072 - CODE_RING * CODE_BYTES) / (p.bpad * 2 * X_ATOM)));
    // The widest split of k whose clusters all run at once.
    p.cs = 1;
    if (pl.d.epi != EPI_HEAD)
        for (int c = std::min(lin::MAX_CLUSTER, p.stages); c > 1; --c)
            if (p.tiles <= active_clusters(ctx, c)) {
                p.cs = c;
                break;
            }
    CUtensorMap tm_w, tm_x;
    if (!encode(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, w.K / 2, w.N, w.K / 2, KS / 2, BM, CU_TENSOR_MAP_SWIZZLE_64B) ||
        !encode(&tm_x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, pl.x, w.K, pl.d.B, pl.ldx * 2, 64, p.bpad, CU_TENSOR_MAP_SWIZZLE_128B))
        return GPT2_B200_EDEVICE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.cs > 1 ? p.tiles * p.cs : std::min(p.tiles, ctx->num_sms)), 1, 1);
    cfg.blockDim = dim3(TC_THREADS, 1, 1);
    cfg.dynamicSmemBytes = TC_SMEM - 1024;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (p.cs > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = static_cast<unsigned>(p.cs);
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    if (pl.pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    return cudaLaunchKernelEx(&cfg, tc_kernel(w), tm_w, tm_x, p) == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace

int prepare(const Plan &pl) {
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    return pl.d.B <= SIMPLE_MAX_B ? GPT2_B200_OK : prepare_tc(ctx);
}

int launch(const Plan &pl, cudaStream_t stream) {
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    return pl.d.B <= SIMPLE_MAX_B ? launch_simple(pl, stream) : launch_tc(ctx, pl, stream);
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
