// w4_linear.cu — products with 4-bit weights: C[b, n] = e(sum_k x[b, k] * value(n, k) + bias[n]) for the B rows of a
// decoding step (the format and the values: w4.cuh).
#include <algorithm>
#include <type_traits>

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

// What an output needs beside its sum.
struct Extra {
    float bias, resid;
};
__device__ __forceinline__ float bias_of(const Dest &d, int n) { return d.bias && n < d.N ? __half2float(d.bias[n]) : 0.0f; }
__device__ __forceinline__ Extra extra_of(const Dest &d, int b, int n) {
    return {bias_of(d, n), d.epi == EPI_RESID ? __half2float(d.resid[b * d.ldr + n]) : 0.0f};
}

// The output of a sum, and its place in the K/V cache if it has one.
__device__ __forceinline__ __half shaped(const Dest &d, float acc, const Extra &e) {
    acc += e.bias;
    if (d.epi == EPI_GELU) acc = gelu_new(acc);
    if (d.epi == EPI_RESID) acc += e.resid;
    return __float2half_rn(acc);
}
__device__ __forceinline__ void to_cache(const Dest &d, int b, int n, __half h) {
    if (d.epi != EPI_QKV || n < d.E) return;
    int m = n - d.E;
    const bool is_v = m >= d.E;
    if (is_v) m -= d.E;
    const int pos = d.d_pos[b];
    if (pos < 0 || pos >= d.maxT)
        atomicOr(d.status, ST_KV_BAD_POS);
    else
        (is_v ? d.v_dst[b] : d.k_dst[b])[(static_cast<long long>(m >> 6) * d.maxT + pos) * 64 + (m & 63)] = h;
}
__device__ __forceinline__ __half put(const Dest &d, int b, int n, float acc, const Extra &e) {
    const __half h = shaped(d, acc, e);
    if (d.out) d.out[b * d.ldo + n] = h;
    to_cache(d, b, n, h);
    return h;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- few rows
// Few rows of x (rows_do): bound by reading and converting the weights. Warps stream codes from global memory into registers, DEPTH steps ahead of their
// use, and feed mma.sync with them; nothing but x goes through shared memory, and nothing in the loop waits for another warp. (Through TMA,
// TMEM and their barriers, a stage of 8 KB of codes takes longer to hand over than to read.)
//   - A step is 16 features x 128 k: lane (g, t) = (lane / 4, lane % 4) holds 32 neighbouring k, 16 bytes, of features g and g + 8.
//     The sum over k may be taken in any order, so 4 of a lane's k serve as its share of each instruction's 16.
//   - A CTA's W warps are WR rows of 16 features x WK = W / WR pieces of k, whose sums are added through shared memory in their order. CTAs
//     stay and take tile after tile: x is there, and the next tile's codes are on their way while a tile's sums are put together.
//   - One CTA per SM: each has all of x, and x costs the L2 0.3 us per MB beside the codes. (Two of 8 warps: 4096 x 4096 at B = 8 13.6 us
//     against 9.6, 8192 x 2048 10.9 against 8.5.) L1 holds the loads in flight: less of it for more shared memory is 10% slower.
// 1 x 8192 x 8192 with least 15.2 us (2.4 TB/s), 8 x 50257 x 768 13.0 us: 5 us of launch and first bytes, then 4 warps per scheduler
// that wait for loads and for their own conversions (IPC 1.65 and 1.80 of 4: 41 and 45% of the issue slots). 1 x 131072 x 4096 73 us (3.9 TB/s).
constexpr int CHUNK = 128;
constexpr int DEPTH = 4;
constexpr int ROWS_MAX_B = 16;
constexpr int MAX_X = 3 << 14;      // elements of x
constexpr int X_BYTES = 2 * (MAX_X + ROWS_MAX_B * 16 * CHUNK) + ROWS_MAX_B * 64;  // in shared memory: rows in whole steps of 16 pieces, half a line more

__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// Volatile, so that a load stays where the registers of the step before become free: moved further up, its result would have to be
// copied, which waits for it.
__device__ __forceinline__ void ld_codes(uint4 &v, const uint8_t *p) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
}
__device__ __forceinline__ void ld_scale(uint32_t &v, const uint8_t *p) { asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v) : "l"(p)); }
// The same, or 0.
__device__ __forceinline__ void ld_scale_if(uint32_t &v, const uint8_t *p, bool in) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %2, 0;\nmov.u32 %0, 0;\n@p ld.global.nc.u16 %0, [%1];\n}" : "=&r"(v) : "l"(p), "r"(static_cast<uint32_t>(in)));
}
// W warps, WR of them side by side; NT instructions of 8 rows each.
template <int W, int WR, int NT, bool LEAST>
__global__ void __launch_bounds__(W * 32, 1) k_w4_rows(const RowParams p) {
    constexpr int WK = W / WR, COLS = 8 * NT, FEATURES = 16 * WR;
    extern __shared__ __align__(16) uint8_t xs[];  // [B][steps * WK * 256 + 64]: x, 16-byte pieces ordered for the loop
    __shared__ float red[2][WK][FEATURES][COLS + 1];
    const Dest &d = p.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int wr = warp % WR, kg = warp / WR;
    const int x_row = p.steps * WK * 256 + 64;  // the odd half line keeps neighbouring rows on different banks

    uint4 qa[DEPTH], qb[DEPTH];
    uint32_t sa[DEPTH], sb[DEPTH], la[DEPTH], lb[DEPTH];
    // A lane's place in a tile: its first codes and scales of feature g, and the way to those of the other feature. Nothing outside is
    // read: features past the last are read as the last and dropped, steps past the last k as the lane's last one (or k = 0) under scales
    // of 0, since x is 0 there and a value may be infinite.
    struct Place {
        const uint8_t *qa, *qb, *sa, *sb;
    };
    const int k_lane = kg * CHUNK + 32 * t;
    const int k_first = k_lane < p.K ? k_lane : 0, last = k_lane < p.K ? (p.K - 1 - k_lane) / (CHUNK * WK) : -1;
    const auto place = [&](int tile) {
        const int n = min(tile * FEATURES + wr * 16 + g, d.N - 1), m = min(tile * FEATURES + wr * 16 + g + 8, d.N - 1);
        const uint8_t *s = reinterpret_cast<const uint8_t *>(p.scale + static_cast<long long>(k_first >> p.shift) * d.N);
        return Place{p.codes + (static_cast<long long>(n) * p.K + k_first) / 2, p.codes + (static_cast<long long>(m) * p.K + k_first) / 2, s + 2ll * n, s + 2ll * m};
    };
    constexpr int Q_STEP = CHUNK * WK / 2;
    const long long s_step = ((CHUNK * WK) >> p.shift) * 2ll * d.N;
    const long long to_least = (p.least - p.scale) * 2;
    const auto fetch = [&](int u, const Place &at, int step) {
        const bool in = step <= last;
        step = in ? step : max(last, 0);
        const long long s = step * s_step;
        ld_codes(qa[u], at.qa + static_cast<long long>(step) * Q_STEP);
        ld_codes(qb[u], at.qb + static_cast<long long>(step) * Q_STEP);
        ld_scale_if(sa[u], at.sa + s, in);
        ld_scale_if(sb[u], at.sb + s, in);
        if (LEAST) {
            ld_scale_if(la[u], at.sa + s + to_least, in);
            ld_scale_if(lb[u], at.sb + s + to_least, in);
        }
    };
    const int full = p.K / (CHUNK * WK);  // steps that are whole for every lane
    int tile = blockIdx.x;
    Place here = place(tile), then = here;
    const auto fetch_first = [&] {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            la[u] = lb[u] = 0;
            fetch(u, here, u);
        }
    };
    const auto fill = [&] {
        const unsigned per = p.steps * WK * 16, all = d.B * per;  // pieces of 8 k per row; zeros behind the last k
        // Each CTA starts elsewhere: all that read the same lines in the same order meet at one part of the L2 after another.
        const unsigned start = (blockIdx.x * 8u * 37u + tid) % all;
        unsigned b = start / per, i = start % per;
        for (unsigned done = tid; done < all; done += W * 32) {
            const int k = i * 8;  // piece i & 15 = 4 t + j of its chunk goes to place 4 j + t
            cp_async16(xs + b * x_row + (i >> 4) * 256 + ((i & 3) * 4 + (i >> 2 & 3)) * 16, p.x + b * p.ldx + min(k, p.K - 8), k < p.K);
            i += W * 32;
            while (i >= per) {
                i -= per;
                if (++b == d.B) b = 0;
            }
        }
    };
    // Behind another kernel the codes go first, since they need not wait for it. Otherwise x does: behind the codes of all CTAs, which
    // fill HBM's queues, it takes 4000 to 8000 cycles to come, without them 1500.
    if (p.ahead) fetch_first();
    grid_dependency_wait();
    grid_launch_dependents();
    fill();
    if (!p.ahead) fetch_first();
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    // Rows of x past the last are read as the last: the columns are dropped.
    const uint8_t *xr[NT];
#pragma unroll
    for (int q = 0; q < NT; ++q) xr[q] = xs + min(8 * q + g, d.B - 1) * x_row + kg * 256 + t * 16;

    // The outputs of this thread: 16 lanes take 16 neighbouring features of a row of x.
    const int sub = tid >> 4, f = tid & 15, units = WR * d.B;
    for (int turn = 0; tile < p.tiles; tile += gridDim.x, turn ^= 1) {
        const int n0 = tile * FEATURES, next = tile + gridDim.x;
        Extra early = {0.0f, 0.0f};
        if (sub < units && n0 + sub % WR * 16 + f < d.N) early = extra_of(d, sub / WR, n0 + sub % WR * 16 + f);
        float c[NT][4] = {};
        if (next < p.tiles) then = place(next);
        int x_at = 0, i0 = 0;
        const auto products = [&](int u, auto any_big) {
            constexpr bool BIG = decltype(any_big)::value;
            const Scale ka = scale_of<LEAST, BIG>(sa[u], la[u]), kb = scale_of<LEAST, BIG>(sb[u], lb[u]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t va[4], vb[4];
                values_of<LEAST, BIG>((&qa[u].x)[j], ka, va);
                values_of<LEAST, BIG>((&qb[u].x)[j], kb, vb);
                const uint32_t a0[4] = {va[0], vb[0], va[1], vb[1]}, a1[4] = {va[2], vb[2], va[3], vb[3]};
#pragma unroll
                for (int q = 0; q < NT; ++q) {
                    const uint4 xv = *reinterpret_cast<const uint4 *>(xr[q] + x_at + u * (WK * 256) + j * 64);
                    mma16816(c[q], a0, xv.x, xv.y);
                    mma16816(c[q], a1, xv.z, xv.w);
                }
            }
        };
        const auto use = [&](int u) {
            if (__any_sync(0xFFFFFFFFu, big_scale(max(sa[u], sb[u]))))
                products(u, std::true_type());
            else
                products(u, std::false_type());
        };
        // Whole rounds whose next fetches are of this tile and all there: no checks, addresses a constant apart.
        if (i0 + 2 * DEPTH <= full) {
            const uint8_t *pa = here.qa + static_cast<long long>(i0 + DEPTH) * Q_STEP, *pb = here.qb + static_cast<long long>(i0 + DEPTH) * Q_STEP;
            const uint8_t *ps = here.sa + (i0 + DEPTH) * s_step;
            const long long other = here.sb - here.sa;
            for (; i0 + 2 * DEPTH <= full; i0 += DEPTH) {
#pragma unroll
                for (int u = 0; u < DEPTH; ++u) {
                    use(u);
                    ld_codes(qa[u], pa + u * Q_STEP);
                    ld_codes(qb[u], pb + u * Q_STEP);
                    ld_scale(sa[u], ps);
                    ld_scale(sb[u], ps + other);
                    if (LEAST) {
                        ld_scale(la[u], ps + to_least);
                        ld_scale(lb[u], ps + to_least + other);
                    }
                    ps += s_step;
                }
                pa += DEPTH * Q_STEP;
                pb += DEPTH * Q_STEP;
                x_at += DEPTH * WK * 256;
            }
        }
        for (; i0 < p.steps; i0 += DEPTH, x_at += DEPTH * WK * 256) {
#pragma unroll
            for (int u = 0; u < DEPTH; ++u) {
                const int i = i0 + u;
                if (i >= p.steps) break;
                use(u);
                if (i + DEPTH < p.steps)
                    fetch(u, here, i + DEPTH);
                else if (next < p.tiles)
                    fetch(u, then, u);
            }
        }
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[turn][kg][wr * 16 + g + 8 * (i >> 1)][8 * q + 2 * t + (i & 1)] = c[q][i];
        here = then;
        __syncthreads();  // the other half of red is free: its readers came here
        for (int unit = sub; unit < (units + 1) / 2 * 2; unit += 2 * W) {
            const int b = unit / WR, n = unit % WR * 16 + f;
            unsigned long long key = 0;
            const bool in = unit < units && n0 + n < d.N;
            if (in) {
                float sum = 0.0f;
#pragma unroll
                for (int q = 0; q < WK; ++q) sum += red[turn][q][n][b];
                const float h = __half2float(put(d, b, n0 + n, sum, unit == sub ? early : extra_of(d, b, n0 + n))) + 0.0f;
                if (h == h) key = lin::argmax_key(h, static_cast<unsigned>(n0 + n));
            }
            if (d.epi == EPI_HEAD) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
                if (in && f == 0) d.amax[static_cast<long long>(b) * d.keys + (n0 + n) / 16] = key;
            }
        }
    }
}

// ---------------------------------------------------------------- many rows
// The rest, on tcgen05: 256 features x up to 128 rows of x per CTA, as two MMAs of 128 features that share x; more rows are
// several column blocks. Sums of 128 k at a time:
//   warp 0       TMA of the codes, 2 x 128 features x 64 bytes (64-byte swizzle), as they lie;
//   warp 2       TMA of x, 128-byte swizzle, K-major: the MMAs' B operand;
//   warps 4-19   two warpgroups per 128 features, at alternate stages: a thread converts the 128 codes of one feature into 64 TMEM
//                columns, the MMA's A operand; they also take the finished tiles out of TMEM, once two stages of the next one are there;
//   warps 1, 3   8 MMAs (K 16) each, from TMEM and shared memory, accumulators in TMEM: one waits while the other's run.
// A hand-over through an mbarrier costs each role 200 to 400 cycles, and HBM delivers the codes of a stage in 700: so a stage is 32768
// codes and each role passes one barrier per stage. Two tiles of features per x halve what x costs the L2: at 128 rows of x, 16 KB
// of codes come with 32 KB of x (one tile of 128 x 256: 8 with 64, 10 TB/s from the L2 and no more).
// 64 x 8192 x 8192 20.0 us (bytes 5.8): 16 stages of 1250 cycles, of which the conversion needs 610 to 800 and the hand-overs the rest, and
// 10 us of launch, start and the cluster's sums; 256 x 16384 x 8192 61 us, 1125 TFLOP/s of the 1680 measured for cuBLAS, by the MMAs and
// their hand-overs.
// A few features and a long k: the CTAs of a cluster share a tile's k and add their sums through distributed shared memory, in rank order.
constexpr int BM = 128;                      // features of an MMA, one TMEM lane each
constexpr int TILES = 2;                     // MMAs side by side
constexpr int FEATURES = BM * TILES;
constexpr int KS = 128;                      // k of a stage
constexpr int CODE_BYTES = FEATURES * KS / 2;
constexpr int CODE_RING = 4;
constexpr int MAX_X_RING = 8;
constexpr int MAX_COLS = 128;                // rows of x per block
constexpr int PUSH_COLS = 64;                // columns up to which the rings leave room for the cluster's sums
constexpr int A_BUFS = 2;                    // converted stages
constexpr int A_COLS = KS / 2;               // TMEM columns of one
constexpr int TC_THREADS = 640;
constexpr int CONVERTERS = 16;               // warps
constexpr size_t TC_SMEM = 226 * 1024;       // the SM for itself: no other CTA's TMEM allocation meets this one's

__device__ __forceinline__ float4 dsmem_ld_v4(uint32_t cluster_saddr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_saddr) : "memory");
    return v;
}
__device__ __forceinline__ void dsmem_st_f32(uint32_t cluster_saddr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_saddr), "f"(v) : "memory");
}

// 16 columns from c on of this warp's 32 features out of TMEM, through the epilogue. acc: the accumulator's first column; n: this lane's
// feature; b0: the block's first row of x. Everything is read before the first output is written: the compiler cannot know that
// an output is no input of the next, and would wait for each.
template <int EPI>
__device__ __forceinline__ void epilogue(const Dest &d, uint32_t acc, int warp4, int lane, int n, int b0, int c) {
    uint32_t r[16];
    tmem_ld16(acc + (static_cast<uint32_t>(warp4 * 32) << 16) + c, r);
    const int first = b0 + c, many = min(16, d.B - first);
    const float bias = bias_of(d, n);
    float resid[16];
    if (EPI == EPI_RESID) {
        const __half *from = d.resid + first * d.ldr + n;
#pragma unroll
        for (int j = 0; j < 16; ++j) resid[j] = j < many && n < d.N ? __half2float(from[j * d.ldr]) : 0.0f;
    }
    tmem_wait_ld();
    __half h[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float v = __uint_as_float(r[j]) + bias;
        if (EPI == EPI_GELU) v = gelu_new(v);
        if (EPI == EPI_RESID) v += resid[j];
        h[j] = __float2half_rn(v);
    }
    if (d.out && n < d.N) {
        __half *out = d.out + first * d.ldo + n;
        if (many == 16) {
#pragma unroll
            for (int j = 0; j < 16; ++j, out += d.ldo) *out = h[j];
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j, out += d.ldo)
                if (j < many) *out = h[j];
        }
    }
    if (EPI == EPI_QKV && n < d.N) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < many) to_cache(d, first + j, n, h[j]);
    }
    if (EPI == EPI_HEAD) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j >= many) break;
            const float v = __half2float(h[j]) + 0.0f;
            const unsigned long long key = n < d.N && v == v ? lin::argmax_key(v, static_cast<unsigned>(n)) : 0ull;
            const unsigned hi = static_cast<unsigned>(key >> 32), mhi = __reduce_max_sync(0xFFFFFFFFu, hi);
            const unsigned mlo = __reduce_max_sync(0xFFFFFFFFu, hi == mhi ? static_cast<unsigned>(key) : 0u);
            if (lane == 0) d.amax[static_cast<long long>(first + j) * d.keys + n / 32] = static_cast<unsigned long long>(mhi) << 32 | mlo;
        }
    }
}

// GS: groups per stage, 128 / group.
template <int GS, bool LEAST>
__global__ void __launch_bounds__(TC_THREADS, 1) k_w4_tc(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const TcParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t c_full[CODE_RING], c_empty[CODE_RING], x_full[MAX_X_RING], x_empty[MAX_X_RING], a_full[TILES][A_BUFS], a_empty[TILES][A_BUFS], acc_full[2],
        acc_empty[2], last_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int bad;  // a wait gave up here, or in a CTA that shares the tile: nothing more is written
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *const x_smem = smem + CODE_RING * CODE_BYTES;
    const int x_bytes = p.bpad * 2 * KS;
    const int rank = static_cast<int>(cluster_rank());
    const int first_tile = blockIdx.x / p.cs, tile_step = gridDim.x / p.cs, b0 = blockIdx.y * p.bpad;
    const int my_tiles = (p.tiles - first_tile + tile_step - 1) / tile_step;
    const int s0 = rank * p.stages / p.cs, ns = (rank + 1) * p.stages / p.cs - s0;  // this CTA's stages of each tile
    const int total = my_tiles * ns;

    // The producers set up their own barriers and start; the others meet behind the allocation.
    const auto code_copy = [&](int slot, int k, int n0) {
        mbar_arrive_expect_tx(&c_full[slot], CODE_BYTES);
#pragma unroll
        for (int w = 0; w < TILES; ++w) tma_load_2d(smem + slot * CODE_BYTES + w * (CODE_BYTES / TILES), &tm_w, &c_full[slot], k / 2, n0 + w * BM);
    };
    // Codes do not depend on the kernel before this one, so nothing waits for it.
    const int early = min(min(total, ns), CODE_RING), early_x = min(min(total, ns), p.x_ring);
    const auto x_copy = [&](int slot, int stage) {
        mbar_arrive_expect_tx(&x_full[slot], static_cast<uint32_t>(x_bytes));
        tma_load_2d(x_smem + slot * x_bytes, &tm_x, &x_full[slot], stage * KS, b0);
        tma_load_2d(x_smem + slot * x_bytes + x_bytes / 2, &tm_x, &x_full[slot], stage * KS + 64, b0);
    };
    if (warp == 0) {
        if (lane < CODE_RING) {
            mbar_init(&c_full[lane], 1);
            mbar_init(&c_empty[lane], CONVERTERS / A_BUFS);
        }
        fence_mbar_init();
        __syncwarp();
        if (elect_one())
            for (int i = 0; i < early; ++i) code_copy(i, (s0 + i) * KS, first_tile * FEATURES);
        __syncwarp();
    } else if (warp == 1) {
        if (lane < TILES * A_BUFS) {
            mbar_init(&a_full[0][lane], 4);
            mbar_init(&a_empty[0][lane], 1);
        }
        if (lane < 2) {
            mbar_init(&acc_full[lane], TILES);
            mbar_init(&acc_empty[lane], CONVERTERS);
        }
        if (lane == 31) mbar_init(&last_full, TILES);
        fence_mbar_init();
        __syncwarp();
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    } else if (warp == 2) {
        if (lane < MAX_X_RING) {
            mbar_init(&x_full[lane], 1);
            mbar_init(&x_empty[lane], TILES);
        }
        fence_mbar_init();
        __syncwarp();
        grid_dependency_wait();
        if (elect_one())
            for (int i = 0; i < early_x; ++i) x_copy(i, s0 + i);
        __syncwarp();
    } else if (tid == 96) {
        bad = 0;
    }
    __syncwarp();
    if (p.cs > 1) cluster_arrive_relaxed();  // waited for before the first write to another CTA
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All of the SM's columns are this CTA's, from 0 on; as constants they cost the MMAs nothing (out of a register, each operand of each
    // MMA is moved to a uniform one).
    constexpr uint32_t tm_a = 0, tm_acc = A_BUFS * TILES * A_COLS;
    grid_launch_dependents();

    bool gave_up = false;  // this warp did (lane 0 knows)
    const auto fail = [&] {
        gave_up = true;
        if (lane == 0) {
            bad = 1;
            atomicOr(p.d.status, ST_LINEAR_TIMEOUT);
        }
    };
    if (tid == 0 && tmem_slot != 0) bad = gave_up = true;  // cannot be
    // Each role counts slots, phases, stages and tiles by hand: one warp's divisions by run-time numbers take longer than a stage.
    if (warp == 0) {
        const bool leader = elect_one();
        int it = early, i = early, n0 = first_tile * FEATURES;
        for (; it < total; ++it) {
            if (i == ns) {
                i = 0;
                n0 += tile_step * FEATURES;
            }
            const int slot = it % CODE_RING;
            const bool ok = it < CODE_RING || mbar_wait(&c_empty[slot], (it / CODE_RING - 1) & 1, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                fail();
                break;
            }
            if (leader) code_copy(slot, (s0 + i) * KS, n0);
            ++i;
            __syncwarp();
        }
        // every copy has landed before this CTA may end, whatever became of the others
        for (int j = max(0, it - CODE_RING); j < it; ++j) mbar_wait(&c_full[j % CODE_RING], (j / CODE_RING) & 1, p.timeout_ns);
    } else {
        grid_dependency_wait();
    }
    if (warp == 2) {
        const bool leader = elect_one();
        int i = early_x, slot = early_x == p.x_ring ? 0 : early_x, at = early_x;
        uint32_t phase = early_x == p.x_ring ? 0 : 1;  // of x_empty: passed at once while the ring fills
        for (; at < total; ++at) {
            if (i == ns) i = 0;
            const bool ok = mbar_wait(&x_empty[slot], phase, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                fail();
                break;
            }
            if (leader) x_copy(slot, s0 + i);
            ++i;
            if (++slot == p.x_ring) {
                slot = 0;
                phase ^= 1;
            }
            __syncwarp();
        }
        for (int j = max(0, at - p.x_ring); j < at; ++j) mbar_wait(&x_full[j % p.x_ring], (j / p.x_ring) & 1, p.timeout_ns);
    }
    if (warp == 1 || warp == 3) {
        const int w = warp >> 1;  // its 128 features
        const bool leader = elect_one();
        const uint32_t idesc = idesc_f16_f32(BM, p.bpad, 0, 0);
        const uint64_t dx = sdesc_sw128(smem_u32(x_smem), 16, 1024);
        const uint32_t x_lo = static_cast<uint32_t>(dx), x_hi = static_cast<uint32_t>(dx >> 32), x_step = static_cast<uint32_t>(x_bytes) >> 4;
        // One flat loop whose only exits are votes: what the MMAs take stays in uniform registers (32 cycles per MMA of 64 columns; 56 with
        // the waits' results carried through nested loops).
        int i = 0, buf = 0, slot = 0, acc = 0;
        uint32_t x_phase = 0, a_phase = 0, acc_phase = 1;  // of acc_empty: passed at once for the first tiles
        bool ok = true;
        for (int it = 0; it < total; ++it) {
            if (i == 0) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_spin(&acc_empty[acc], acc_phase, p.timeout_ns));
                if (!ok) break;
            }
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_spin(&x_full[slot], x_phase, p.timeout_ns));
            if (!ok) break;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_spin(&a_full[w][buf], a_phase, p.timeout_ns));
            if (!ok) break;
            tc_fence_after();
            const uint32_t b_lo = x_lo + static_cast<uint32_t>(slot) * x_step, from = tm_a + (buf * TILES + w) * A_COLS, to = tm_acc + (acc * TILES + w) * p.bpad;
            if (leader) {
                umma_f16_ts_lohi(to, from, b_lo, x_hi, idesc, i > 0 ? 1u : 0u);
#pragma unroll
                for (int kk = 1; kk < KS / 16; ++kk) umma_f16_ts_lohi(to, from + kk * 8, b_lo + kk / 4 * (x_step / 2) + kk % 4 * 2, x_hi, idesc, 1u);
                umma_commit(&a_empty[w][buf]);
                umma_commit(&x_empty[slot]);
                if (i == ns - 1) umma_commit(&acc_full[acc]);
            }
            __syncwarp();
            buf ^= 1;
            if (buf == 0) a_phase ^= 1;
            if (++slot == p.x_ring) {
                slot = 0;
                x_phase ^= 1;
            }
            if (++i == ns) {
                i = 0;
                if (++acc == p.nacc) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
        }
        if (!ok) fail();
        __syncwarp();
        if (leader) umma_commit(&last_full);  // arrives when all that was issued is done
    }
    // Sums that another CTA of the cluster adds: pushed into a buffer of its own there, or left where the rings were.
    const uint32_t parts = smem_u32(smem) + (p.push ? CODE_RING * CODE_BYTES + p.x_ring * x_bytes : 0);
    if (warp >= 4) {
        const int wg = (warp - 4) >> 2, warp4 = warp & 3, row = warp4 * 32 + lane;
        const int tile_w = wg & 1, turn = wg >> 1;  // its 128 features; its stages are the even or the odd ones, in A buffer `turn`
        const uint32_t lanes = static_cast<uint32_t>(warp4 * 32) << 16;
        const uint32_t to = tm_a + lanes + (turn * TILES + tile_w) * A_COLS;
        const uint8_t *from = smem + tile_w * (CODE_BYTES / TILES) + row * 64;
        // Scales are fetched for the warpgroup's next stage, two ahead, when this one's have been used.
        __half sc[GS], lo[GS];
        int si = turn, sn = first_tile * FEATURES + tile_w * BM + row;  // stage of the tile, and feature, of the next
        const auto scales = [&] {
            while (si >= ns) {
                si -= ns;
                sn += tile_step * FEATURES;
            }
#pragma unroll
            for (int q = 0; q < GS; ++q) {
                const int k = (s0 + si) * KS + q * (KS / GS);
                const bool in = sn < p.d.N && k < p.K;
                const long long at = static_cast<long long>(k >> p.shift) * p.d.N + sn;
                sc[q] = in ? p.scale[at] : __float2half_rn(0.0f);
                if (LEAST) lo[q] = in ? p.least[at] : __float2half_rn(0.0f);
            }
            si += 2;
        };
        // Takes tile j out of TMEM; the pieces of 16 columns of its two accumulators are shared by the warpgroups.
        int taken = 0;
        const auto take = [&] {
            const int j = taken++, acc = p.nacc == 2 ? j & 1 : 0, round = p.nacc == 2 ? j >> 1 : j, n0 = (first_tile + j * tile_step) * FEATURES;
            const bool ok = j == my_tiles - 1 ? mbar_wait(&last_full, 0, p.timeout_ns) : mbar_wait(&acc_full[acc], round & 1, p.timeout_ns);
            if (!__all_sync(0xFFFFFFFFu, ok)) fail();
            __syncwarp();
            if (*reinterpret_cast<volatile int *>(&bad)) return;
            tc_fence_after();
            const int per = p.bpad / 16;
            for (int piece = turn; piece < per; piece += 2) {
                const int c = piece * 16, f = tile_w * BM + row;
                const uint32_t at = tm_acc + (acc * TILES + tile_w) * p.bpad;
                if (p.cs == 1) {
                    switch (p.d.epi) {
                        case EPI_STORE: epilogue<EPI_STORE>(p.d, at, warp4, lane, n0 + f, b0, c); break;
                        case EPI_GELU: epilogue<EPI_GELU>(p.d, at, warp4, lane, n0 + f, b0, c); break;
                        case EPI_RESID: epilogue<EPI_RESID>(p.d, at, warp4, lane, n0 + f, b0, c); break;
                        case EPI_QKV: epilogue<EPI_QKV>(p.d, at, warp4, lane, n0 + f, b0, c); break;
                        default: epilogue<EPI_HEAD>(p.d, at, warp4, lane, n0 + f, b0, c);
                    }
                } else {
                    uint32_t r[16];
                    tmem_ld16(at + lanes + c, r);
                    tmem_wait_ld();
                    if (p.push) {
                        int q = c / p.share, left = (q + 1) * p.share - c;  // the CTA that adds column c, and its columns from there on
                        uint32_t there = dsmem_addr(parts + ((rank * p.share + p.share - left) * FEATURES + f) * 4, static_cast<uint32_t>(q));
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            dsmem_st_f32(there, __uint_as_float(r[i]));
                            there += FEATURES * 4;
                            if (--left == 0) {
                                left = p.share;
                                there = dsmem_addr(parts + (rank * p.share * FEATURES + f) * 4, static_cast<uint32_t>(min(++q, p.cs - 1)));
                            }
                        }
                    } else {
                        float *part = reinterpret_cast<float *>(smem);
#pragma unroll
                        for (int i = 0; i < 16; ++i) part[(c + i) * FEATURES + f] = __uint_as_float(r[i]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[acc]);
        };
        scales();
        bool ok = true;
        int due = ns + 2;  // from this stage on the first tile is taken: it is converted, and two stages of the next
        uint32_t a_phase = 1;  // of a_empty: passed at once for the first stage
        for (int it = turn; it < total; it += 2) {
            while (it >= due) {
                take();
                due += ns;
            }
            const int slot = it % CODE_RING;
            ok = mbar_wait(&c_full[slot], (it / CODE_RING) & 1, p.timeout_ns);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            const uint8_t *st = from + slot * CODE_BYTES;
            uint4 codes[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) codes[q] = *reinterpret_cast<const uint4 *>(st + ((q ^ (row >> 1 & 3)) << 4));  // 32 k: the 64-byte swizzle's place
            bool large = false;
#pragma unroll
            for (int q = 0; q < GS; ++q) large = large || big_scale(__half_as_ushort(sc[q]));
            const auto convert = [&](auto any_big) {
                constexpr bool BIG = decltype(any_big)::value;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[32];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int g = (2 * h + q) * GS / 4;
                        const uint4 &w = codes[2 * h + q];
                        const Scale k = scale_of<LEAST, BIG>(__half_as_ushort(sc[g]), LEAST ? __half_as_ushort(lo[g]) : 0);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t four[4];
                            values_of<LEAST, BIG>((&w.x)[j], k, four);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[q * 16 + j * 4 + e] = four[e];
                        }
                    }
                    if (h == 0) {  // half a stage is converted before its buffer has to be free
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&a_empty[tile_w][turn], a_phase, p.timeout_ns));
                        if (!ok) return;
                        tc_fence_after();
                    }
                    tmem_st32(to + h * 32, v);
                }
            };
            if (__any_sync(0xFFFFFFFFu, large))
                convert(std::true_type());
            else
                convert(std::false_type());
            if (!ok) break;
            a_phase ^= 1;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&a_full[tile_w][turn]);
                mbar_arrive(&c_empty[slot]);
            }
            if (it + 2 < total) scales();
        }
        if (!ok) fail();
        __syncwarp();
        if (p.cs > 1) cluster_wait();
        while (taken < my_tiles && !*reinterpret_cast<volatile int *>(&bad)) take();
    } else {
        __syncwarp();
        if (p.cs > 1) cluster_wait();
    }
    // A CTA that gave up left no sums, or not all: the others may not add them. (Kept in a register: every warp's look at `bad` here
    // takes 0.1 us.)
    if (__builtin_expect(gave_up, 0) && p.cs > 1 && lane == 0) {
#pragma unroll 1
        for (int q = 0; q < p.cs; ++q) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dsmem_addr(smem_u32(&bad), static_cast<uint32_t>(q))), "r"(1) : "memory");
    }
    __syncwarp();
    if (p.cs > 1) {
        // Every CTA of the cluster has `share` of the columns, and adds them over the ranks in their order: 4 features a thread.
        const int f = tid % (FEATURES / 4) * 4, n = first_tile * FEATURES + f, c0 = rank * p.share + tid / (FEATURES / 4);
        const int c1 = min(min(p.d.B - b0, p.bpad), (rank + 1) * p.share);
        float bias[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = bias_of(p.d, n + i);
        cluster_sync_all();
        for (int c = c0; c < c1; c += TC_THREADS / (FEATURES / 4)) {
            const int b = b0 + c;
            float4 v[lin::MAX_CLUSTER];
#pragma unroll
            for (int q = 0; q < lin::MAX_CLUSTER; ++q) {
                if (q >= p.cs) break;
                v[q] = p.push ? lds_v4(parts + ((q * p.share + c - rank * p.share) * FEATURES + f) * 4)
                              : dsmem_ld_v4(dsmem_addr(parts + (c * FEATURES + f) * 4, static_cast<uint32_t>(q)));
            }
            float resid[4] = {};
            if (p.d.epi == EPI_RESID) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.d.N) resid[i] = __half2float(p.d.resid[b * p.d.ldr + n + i]);
            }
            float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int q = 1; q < lin::MAX_CLUSTER; ++q) {
                if (q >= p.cs) break;
                sum[0] += v[q].x;
                sum[1] += v[q].y;
                sum[2] += v[q].z;
                sum[3] += v[q].w;
            }
            if (*reinterpret_cast<volatile int *>(&bad)) break;
            __half h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = shaped(p.d, sum[i], {bias[i], resid[i]});
            __half *out = p.d.out + b * p.d.ldo + n;
            if (n + 3 < p.d.N && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
                *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(h);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.d.N) out[i] = h[i];
            }
            if (p.d.epi == EPI_QKV)
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.d.N) to_cache(p.d, b, n + i, h[i]);
        }
        if (!p.push) cluster_sync_all();  // the others may still be reading this CTA's sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_slot, 512);
}

typedef void (*TcKernel)(CUtensorMap, CUtensorMap, TcParams);
template <bool LEAST>
TcKernel tc_kernel(int group) {
    return group == 128 ? k_w4_tc<1, LEAST> : group == 64 ? k_w4_tc<2, LEAST> : k_w4_tc<4, LEAST>;
}
// Which of the two. k_w4_rows copies all of x into every SM and has instructions of 8 columns, k_w4_tc takes 3 us to start and
// then does not mind the rows. us, rows against tcgen05: 2304 x 768 4.7 against 6.4 at B = 1, 5.3 against 6.6 at 8, 6.1 against 6.6 at 16;
// 768 x 4 * 768 7.7 against 7.7 at 16; 4096 x 1024 6.7 against 7.1 at 16; 50257 x 768 11.0 against 13.8 at 1, 13.0 against 13.9 at 8, but 15.0
// against 13.8 at 9; 8192 x 2048 9.5 against 9.2 at 9; 4096 x 4096 7.5 against 10.0 at 1, 9.6 against 10.2 at 8; 8192 x 8192 15.4 against
// 17.9 at 1, 16.8 at 4, and with 96 KB of x and more 19.0 against 17.9 at 6. A decode step of 9 sequences 300 against 377, of 16 370 against 387.
bool rows_do(int B, int N, int K) {
    const long long x = static_cast<long long>(B) * K, weight = static_cast<long long>(N) * K;
    return (B <= 8 && x <= 1 << 15) || (B <= ROWS_MAX_B && x <= MAX_X && weight <= 1 << 22);
}

typedef void (*RowKernel)(RowParams);
template <int NT, bool LEAST>
RowKernel row_kernel(int warps, int wr) {
    if (warps == 8) return k_w4_rows<8, 1, NT, LEAST>;
    if (NT == 1 && wr == 1) return k_w4_rows<16, 1, 1, LEAST>;
    return wr == 2 ? k_w4_rows<16, 2, NT, LEAST> : wr == 4 ? k_w4_rows<16, 4, NT, LEAST> : wr == 8 ? k_w4_rows<16, 8, NT, LEAST> : k_w4_rows<16, 16, NT, LEAST>;
}
RowKernel row_kernel(int B, bool least, int warps, int wr) {
    return B <= 8 ? (least ? row_kernel<1, true>(warps, wr) : row_kernel<1, false>(warps, wr))
                  : (least ? row_kernel<2, true>(warps, wr) : row_kernel<2, false>(warps, wr));
}

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

// The kernels' shared memory, on the current device once: so that neither a launch nor a capture has to.
int prepare(DeviceContext *ctx) {
    if (ctx->w4_attr_done) return GPT2_B200_OK;
    RelaxedCapture relaxed;
    for (int wr = 0; wr <= 16; wr = wr ? 2 * wr : 1)  // 0: of 8 warps
        for (int i = wr == 1 ? 1 : 0; i < 4; i += wr == 1 ? 2 : 1)
            if (cudaFuncSetAttribute(row_kernel(i & 1 ? 1 : ROWS_MAX_B, i & 2, wr ? 16 : 8, wr), cudaFuncAttributeMaxDynamicSharedMemorySize, X_BYTES) !=
                cudaSuccess)
                return GPT2_B200_ECUDA;
    for (int group = 32; group <= 128; group *= 2)
        for (const TcKernel k : {tc_kernel<false>(group), tc_kernel<true>(group)})
            if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(TC_SMEM)) != cudaSuccess) return GPT2_B200_ECUDA;
    ctx->w4_attr_done = true;
    return GPT2_B200_OK;
}

// How many clusters of cs CTAs run at once (one CTA per SM), asked once per device.
int active_clusters(DeviceContext *ctx, int cs) {
    int &n = ctx->w4_clusters[cs];
    if (n) return n;
    RelaxedCapture relaxed;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(cs) * 64, 1, 1);
    cfg.blockDim = dim3(TC_THREADS, 1, 1);
    cfg.dynamicSmemBytes = TC_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cs);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, tc_kernel<false>(128), &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n = got;
}

int plan_rows(DeviceContext *ctx, Plan *pl, const GPT2W4 &w, const __half *x, long long ldx) {
    const int B = pl->d.B, chunks = (w.K + CHUNK - 1) / CHUNK, sms = ctx->num_sms;
    RowParams &p = pl->rows;
    p.codes = static_cast<const uint8_t *>(w.codes);
    p.scale = w.scale;
    p.least = w.least;
    p.K = w.K;
    p.shift = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    p.x = x;
    p.ldx = ldx;
    // 8 warps where every tile of 16 features has an SM, which all take a piece of k each. Else 16, and the tile height with the fewest steps
    // of the busiest CTA, a tile's end counted as one. us, 8 against 16 warps at B = 1: 768 x 768 3.2 against 4.0, 768 x 4 * 768 4.4 against
    // 5.1, but 4096 x 1024 6.2 (two CTAs per SM, each with its x) against 5.2.
    const int warps = (w.N + 15) / 16 <= sms ? 8 : 16;
    int wr = 0;
    long long best = 0;
    // (More than 8 rows of weights that small never have so many k that 16 warps would share them.)
    for (int h = warps == 16 && B > 8 ? 2 : 1; h <= (warps == 8 ? 1 : warps); h *= 2) {
        const long long tiles = (static_cast<long long>(w.N) + 16 * h - 1) / (16 * h), rounds = (tiles + sms - 1) / sms;
        const int wk = warps / h, steps = (chunks + wk - 1) / wk;
        const long long cost = rounds * (steps + 1);
        if (wr && cost >= best) continue;
        best = cost;
        wr = h;
        p.tiles = static_cast<int>(tiles);
        p.steps = steps;
    }
    pl->grid = dim3(static_cast<unsigned>(std::min(p.tiles, sms)), 1, 1);
    pl->threads = warps * 32;
    pl->smem = static_cast<size_t>(B) * (p.steps * (warps / wr) * 256 + 64);
    pl->kernel = reinterpret_cast<const void *>(row_kernel(B, w.least != nullptr, warps, wr));
    return GPT2_B200_OK;
}

int plan_tc(DeviceContext *ctx, Plan *pl, const GPT2W4 &w, const __half *x, long long ldx) {
    const Dest &d = pl->d;
    TcParams &p = pl->tc;
    p.scale = w.scale;
    p.least = w.least;
    p.K = w.K;
    p.shift = w.group == 32 ? 5 : w.group == 64 ? 6 : 7;
    p.stages = (w.K + KS - 1) / KS;
    p.tiles = (w.N + FEATURES - 1) / FEATURES;
    // Column blocks and CTAs per tile, by the cycles that they take in a model that is near enough to choose by: 3300 to the first codes, 1000
    // a stage (or the MMAs, 8 a column), 2000 and 90 a column for the sums of a cluster, 40 a column for a tile's outputs without one. (Seen
    // at 64 columns and 1965 MHz: 1250 a stage, and a cluster's sums take 4600 to 4800 longer than outputs without, 8192 x 8192 against
    // 32768 x 2048.) Blocks read the weights
    // again, from the L2, and convert them again, on SMs that have nothing else to do: with a few features and a short k that is
    // cheaper than adding wide sums (64 x 2304 x 768).
    int blocks = 0;
    long long best = 0;
    for (int n = (d.B + MAX_COLS - 1) / MAX_COLS; n <= (d.B + 15) / 16; ++n) {
        const int cols = ((d.B + n - 1) / n + 15) / 16 * 16;
        if ((d.B + cols - 1) / cols != n) continue;  // an empty block
        const long long stage = std::max(1000, 8 * cols);
        for (int c = 1; c <= std::min(lin::MAX_CLUSTER, p.stages); ++c) {
            if (c > 1 && (d.epi == EPI_HEAD || p.tiles > active_clusters(ctx, c) / n)) continue;
            const long long each = std::max(1, ctx->num_sms / n), rounds = c > 1 ? 1 : (p.tiles + each - 1) / each;
            const long long cost = 3300 + rounds * ((p.stages + c - 1) / c * stage + (c > 1 ? 2000 + 90 * cols : 40 * cols));
            if (!blocks || cost < best) {
                best = cost;
                blocks = n;
                p.cs = c;
                p.bpad = cols;
            }
        }
    }
    p.nacc = p.bpad <= 64 ? 2 : 1;
    p.timeout_ns = wait_timeout_ns();
    p.share = (p.bpad + p.cs - 1) / p.cs;
    p.push = p.cs > 1 && p.bpad <= PUSH_COLS;
    const size_t rest = TC_SMEM - 1024 - CODE_RING * CODE_BYTES - (p.push ? static_cast<size_t>(p.cs) * p.share * FEATURES * 4 : 0);
    p.x_ring = std::min<int>(MAX_X_RING, static_cast<int>(rest / (p.bpad * 2 * KS)));
    if (!encode(&pl->tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, w.K / 2, w.N, w.K / 2, KS / 2, BM, CU_TENSOR_MAP_SWIZZLE_64B) ||
        !encode(&pl->tm_x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, w.K, d.B, ldx * 2, 64, p.bpad, CU_TENSOR_MAP_SWIZZLE_128B))
        return GPT2_B200_EDEVICE;
    pl->cluster = p.cs;
    pl->grid = dim3(static_cast<unsigned>(p.cs > 1 ? p.tiles * p.cs : std::min(p.tiles, std::max(1, ctx->num_sms / blocks))), blocks, 1);
    pl->threads = TC_THREADS;
    pl->smem = TC_SMEM;
    pl->kernel = reinterpret_cast<const void *>(w.least ? tc_kernel<true>(w.group) : tc_kernel<false>(w.group));
    return GPT2_B200_OK;
}

}  // namespace

int plan(Plan *pl, int epi, const GPT2W4 &w, const __half *x, long long ldx, int B, const __half *bias, __half *out, long long ldo, const __half *resid, long long ldr) {
    if (!weight_ok(&w) || !x || (reinterpret_cast<uintptr_t>(x) & 15) || (ldx & 7) || ldx < w.K || B < 1 || B > lin::MAX_BPAD) return GPT2_B200_EINVAL;
    if (epi < EPI_STORE || epi > EPI_HEAD || (epi != EPI_HEAD && !out) || (out && ldo < w.N) || (epi == EPI_RESID && (!resid || ldr < w.N)) ||
        ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(resid)) & 1))
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    const int rc = prepare(ctx);
    if (rc != GPT2_B200_OK) return rc;
    *pl = Plan{};
    pl->d.epi = epi;
    pl->d.B = B;
    pl->d.N = w.N;
    pl->d.bias = bias;
    pl->d.out = out;
    pl->d.ldo = ldo;
    pl->d.resid = resid;
    pl->d.ldr = ldr;
    pl->few = rows_do(B, w.N, w.K);
    pl->d.keys = pl->few ? (w.N + 15) / 16 : (w.N + FEATURES - 1) / FEATURES * (FEATURES / 32);
    pl->d.status = ctx->status;
    pl->cluster = 1;
    return pl->few ? plan_rows(ctx, pl, w, x, ldx) : plan_tc(ctx, pl, w, x, ldx);
}

int launch(const Plan &pl, const Dest &d, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = pl.grid;
    cfg.blockDim = dim3(pl.threads, 1, 1);
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (pl.cluster > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = static_cast<unsigned>(pl.cluster);
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
    cudaError_t err;
    if (pl.few) {
        RowParams p = pl.rows;
        p.d = d;
        p.ahead = pl.pdl;
        void *args[1] = {&p};
        err = cudaLaunchKernelExC(&cfg, pl.kernel, args);
    } else {
        TcParams p = pl.tc;
        p.d = d;
        void *args[3] = {const_cast<CUtensorMap *>(&pl.tm_w), const_cast<CUtensorMap *>(&pl.tm_x), &p};
        err = cudaLaunchKernelExC(&cfg, pl.kernel, args);
    }
    return err == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace w4
}  // namespace b200

using namespace b200;

extern "C" int gpt2_w4_linear_b200(gpt2_half *C, long long ldc, const gpt2_half *A, long long lda, const GPT2W4 *w, const gpt2_half *bias, const gpt2_half *R,
                                   long long ldr, int B, int epi, cudaStream_t stream) {
    if (!w || !C || epi < GPT2_B200_LINEAR_STORE || epi > GPT2_B200_LINEAR_RESID) return GPT2_B200_EINVAL;
    const int e = epi == GPT2_B200_LINEAR_STORE ? lin::EPI_STORE : epi == GPT2_B200_LINEAR_GELU ? lin::EPI_GELU : lin::EPI_RESID;
    w4::Plan pl;
    const int rc = w4::plan(&pl, e, *w, A, lda, B, bias, C, ldc, e == lin::EPI_RESID ? R : nullptr, ldr);
    return rc == GPT2_B200_OK ? w4::launch(pl, stream) : rc;
}
