// kv8_attend.cu — attention over the paged 8-bit cache.
//
// out = softmax(q K^T / sqrt(D)) V with K = code * scale per block of keys: the scale is constant over a
// block, so it multiplies a key's score (K) and its probability (V), never the D elements. Online
// softmax in base 2: m, l and o are rescaled by 2^(m_old - m_new) when a row's maximum grows.
//
// A decode step reads 2 D + 8 / block bytes per key and K/V head once and does 4 D flops per key and query:
// HBM-bound, if the codes get into the tensor cores cheaply. So:
//   - the products are mma.m16n8k16 in fp16 with fp32 sums. A code is exact in fp16 and so is q; p is not, and goes
//     in as hi + lo (two fp16, 22 bits): rounding it to one fp16 alone would add an error of the size of the
//     output's own rounding. With at most 8 query rows (the decode step) the MMA's rows 8..15 are
//     free and take lo; with 9 to 16 rows lo is a second MMA. mma.sync's rate is far above what HBM feeds
//     (32 MMAs per 4 KB of codes).
//   - a warp takes CK keys at a time (32 for D 64, 16 for D 128: 4 KB of K and V) through a ring of its own in shared
//     memory (cp.async, STAGES - 1 chunks in flight, no CTA barrier). The sum over dims (QK) may run in any order of dims,
//     so a thread's 16 neighbouring code bytes of one key are its operands for 4 k-steps; PV's sum over keys and its
//     column order are as free, so a thread reads 8 or 16 neighbouring dims of the 4 keys whose p it holds, and ends with
//     16 neighbouring output dims. The 16-byte granules of a chunk are permuted so that neither read has bank conflicts.
//   - a lane looks up the page and the two scales of one 16-key granule for the warp, 32 granules at a time, and
//     shuffles hand them out.
//   - p * vscale would leave fp16's range for small scales, so p * (vscale / S) goes in, S the largest
//     vscale the warp has met; o is kept in units of S.
// A CTA is 4 warps on one (row, K/V head, tile of 16 query rows, span of keys): the warps take chunks in turn and are
// merged in shared memory; spans (few rows, long contexts) through the work area by the last CTA to arrive, in span order.
#include "kv8.cuh"
#include "ptx.cuh"

namespace b200 {
namespace kv8 {

constexpr int NW = 4;                // warps per CTA
constexpr int MAX_SPLIT_CTAS = 2048; // grid of a launch that splits keys, at most

int attend_max_ctas() { return MAX_SPLIT_CTAS; }

struct AttParams {
    const __half *q;
    __half *out;
    long long q_row, q_tok, o_row, o_tok;
    const int *d_first, *d_count;
    long long page_stride;  // bytes from a page to the next
    long long k_off, v_off; // from a page's start to this layer's K / V runs of head 0
    float *part;
    unsigned *arrive;
    int L, G, Tq, count, max_len;
    int qtiles, nsplit, span;  // span: keys per split, a multiple of NW * CK
    float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Two int8 codes (as code + 128) in bytes 0, 2 over 0x64 bytes are the halves 1024 + code + 128: exact.
__device__ __forceinline__ uint32_t sub1152(uint32_t h) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2(uint32_t two) {
    uint32_t r;
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
// Four neighbouring codes -> their halves, as two packed pairs.
template <int KIND>
__device__ __forceinline__ void halves4(uint32_t w, uint32_t &h01, uint32_t &h23) {
    if (KIND == GPT2_KV8_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        h01 = sub1152(__byte_perm(u, 0x64646464u, 0x4140));
        h23 = sub1152(__byte_perm(u, 0x64646464u, 0x4342));
    } else {
        h01 = e4m3x2(w);
        h23 = e4m3x2(w >> 16);
    }
}
// Codes of the same four dims of two keys -> per dim the pair (key a, key b).
template <int KIND>
__device__ __forceinline__ void pairs4(uint32_t a, uint32_t b, uint32_t (&h)[4]) {
    halves4<KIND>(__byte_perm(a, b, 0x5140), h[0], h[1]);
    halves4<KIND>(__byte_perm(a, b, 0x7362), h[2], h[3]);
}
__device__ __forceinline__ uint32_t pack_hi(float a, float b, float &la, float &lb) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    la = a - f.x;
    lb = b - f.y;
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// A warp's chunk of CK keys in shared memory: 2 KB of K rows, then 2 KB of V rows, in 16-byte granules.
// Reads: K, a quarter warp takes granules 0..3 (then 4..7 for D 128) of two neighbouring rows; V, a half warp takes two
// granules (8 bytes a lane) or a quarter warp two granules (16 bytes a lane) of rows 0, 2, 4, 6 of an 8-row
// group. The maps put each such set on 8 different bank groups (granule index mod 8).
template <int D>
struct Chunk {
    static constexpr int CK = 2048 / D, GR = CK / 16, ROWG = D / 16;  // granules per row
    __device__ static int k_at(int row, int gr) { return row * ROWG + (D == 64 ? gr : gr ^ ((row & 1) << 2)); }
    __device__ static int v_at(int row, int gr) {
        if (D == 64) {  // 8-row groups: row bits (b2 b1 b0) stored as (b2 b0 b1); the granule's high bit flipped by b2
            const int at = (row & ~3) | ((row & 1) << 1) | ((row >> 1) & 1);
            return at * ROWG + (gr ^ ((row >> 1) & 2));
        }
        return row * ROWG + (gr ^ (row & 6));
    }
};
constexpr int CHUNK_BYTES = 4096;
// Chunks per warp's ring. Three CTAs of 4 x 4 chunks (192 KB) fill an SM's shared memory.
constexpr int STAGES = 4;
constexpr int RING_BYTES = NW * STAGES * CHUNK_BYTES;

template <int KIND, int D, int ROWS>
__global__ void __launch_bounds__(32 * NW, ROWS == 8 && D == 64 ? 3 : 2) k_kv8_attend(const View c, const AttParams a) {
    using C = Chunk<D>;
    constexpr int CK = C::CK, GR = C::GR, NT = CK / 8, KS = D / 16, DT = D / 8, RR = ROWS / 8;
    constexpr int SET = 32 / GR;  // chunks whose granules one look-up covers
    extern __shared__ __align__(128) uint8_t ring_all[];
    float (*so)[ROWS][D + 4] = reinterpret_cast<float (*)[ROWS][D + 4]>(ring_all);  // [NW], behind the main loop
    static_assert(NW * ROWS * (D + 4) * 4 <= RING_BYTES, "the warps' rows fit in the rings");
    __shared__ float sm[NW][ROWS], sl[NW][ROWS];
    __shared__ int is_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.nsplit;
    int unit = blockIdx.x / a.nsplit;
    const int h = unit % c.nHead;
    unit /= c.nHead;
    const int qt = unit % a.qtiles, r = unit / a.qtiles;
    const int R = a.G * a.Tq;

    int n = c.len[r] + (a.d_count ? a.d_count[r] : a.count);
    if (n < 0 || n > a.max_len) {
        if (threadIdx.x == 0 && split == 0 && h == 0 && qt == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        n = 0;
    }
    const int first = a.d_first ? max(a.d_first[r], 0) : 0;
    // keys that some row of the tile sees: [first, last_end); rows of one token see the same
    const int last_row = min(qt * ROWS + ROWS, R) - 1;
    const int last_end = n - a.Tq + last_row / a.G + 1, first_end = n - a.Tq + qt * ROWS / a.G + 1;
    const int base = first & ~(CK - 1);
    const int total = last_end > first ? last_end - base : 0;
    const int active = (total + a.span - 1) / a.span;  // splits with keys
    if (split >= max(active, 1)) return;
    const int lo = base + split * a.span, hi = min(lo + a.span, last_end);
    const int chunks = total ? (hi - lo + CK - 1) / CK : 0;

    // q: thread (g, t) holds dims 64 * (s / 4) + 16 t + 4 (s % 4) .. + 3 of row g (and g + 8) for k-step s
    uint32_t qa[KS][2 * RR];
    int end[RR];
#pragma unroll
    for (int rr = 0; rr < RR; ++rr) {
        const int i = qt * ROWS + g + 8 * rr;
        const bool ok = i < R;
        const int tok = ok ? i / a.G : 0;
        end[rr] = ok ? n - a.Tq + tok + 1 : 0;
        const __half *qp = a.q + r * a.q_row + tok * a.q_tok + static_cast<long long>(h * a.G + (i - tok * a.G)) * D + 16 * t;
#pragma unroll
        for (int s4 = 0; s4 < KS / 4; ++s4) {
            uint4 x[2] = {};
            if (ok) {
                x[0] = *reinterpret_cast<const uint4 *>(qp + 64 * s4);
                x[1] = *reinterpret_cast<const uint4 *>(qp + 64 * s4 + 8);
            }
            const uint32_t *w = reinterpret_cast<const uint32_t *>(x);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                qa[4 * s4 + s][rr] = w[2 * s];
                qa[4 * s4 + s][RR + rr] = w[2 * s + 1];
            }
        }
    }

    float o[DT][4];
#pragma unroll
    for (int j = 0; j < DT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[RR], l[RR], S = 0.0f, invS = 0.0f;
#pragma unroll
    for (int rr = 0; rr < RR; ++rr) m[rr] = -INFINITY, l[rr] = 0.0f;

    // this lane's granule of the current set: its page's byte offset and its scales
    long long goff = 0;
    float gks = 0.0f, gvs = 0.0f;
    unsigned gok = 0;
    bool bad = false;
    auto look_up = [&](int set) {
        const int pos = lo + ((set * SET + lane / GR) * NW + warp) * CK + (lane % GR) * 16;
        int ok = pos < hi && pos + 16 > first;
        if (ok) {
            const int p = c.table[static_cast<long long>(r) * c.maxPages + (pos >> c.page_shift)];
            if (p < 0 || p >= c.nPages) {
                bad = true;
                ok = 0;
            } else {
                const int ip = pos & (c.page - 1), nb = c.page >> c.block_shift;
                const long long run = c.run(p, a.L, 0, h);
                gks = c.scale[run * nb + (ip >> c.block_shift)] * a.scale_log2;
                gvs = c.scale[(run + c.nHead) * nb + (ip >> c.block_shift)];
                goff = p * a.page_stride + static_cast<long long>(h << c.page_shift) * D + ip * D;
            }
        }
        if (!ok) gks = gvs = 0.0f;
        gok = __ballot_sync(0xFFFFFFFFu, ok);
    };
    uint8_t *ring = ring_all + warp * STAGES * CHUNK_BYTES;
    const uint32_t ring_s = smem_u32(ring);
    // A copy instruction of the warp takes 512 bytes: 8 rows (D 64) or 4. V's rows are dealt to the lanes so that its
    // stores, too, meet 8 bank groups per 8 lanes.
    const int krow = lane / C::ROWG;
    const int vrow = D == 64 ? ((lane >> 2) & 1) * 2 + ((lane >> 3) & 1) + (lane >> 4) * 4 : krow;
    const int cgr = lane & (C::ROWG - 1);
    constexpr int CR = 32 / C::ROWG;  // rows per copy instruction
    auto load = [&](int i, int stage) {  // chunk i of this warp; its set has been looked up
        const uint32_t dst = ring_s + stage * CHUNK_BYTES;
#pragma unroll
        for (int gi = 0; gi < GR; ++gi) {
            const int src_lane = (i % SET) * GR + gi;
            const long long off = __shfl_sync(0xFFFFFFFFu, goff, src_lane);
            if (!((gok >> src_lane) & 1u)) continue;
            const uint8_t *kp = c.data + a.k_off + off + krow * D + cgr * 16;
            const uint8_t *vp = c.data + a.v_off + off + vrow * D + cgr * 16;
#pragma unroll
            for (int x = 0; x < 16 / CR; ++x) {
                const int row = gi * 16 + x * CR;
                cp_async16(dst + C::k_at(row + krow, cgr) * 16, kp + x * CR * D);
                cp_async16(dst + 2048 + C::v_at(row + vrow, cgr) * 16, vp + x * CR * D);
            }
        }
    };
    auto compute = [&](const uint8_t *buf, int pos, float (&ks)[GR], float (&vs)[GR], unsigned ok) {
        const uint4 *kb = reinterpret_cast<const uint4 *>(buf), *vb = reinterpret_cast<const uint4 *>(buf + 2048);
        float s[NT][4];
#pragma unroll
        for (int tile = 0; tile < NT; ++tile) s[tile][0] = s[tile][1] = s[tile][2] = s[tile][3] = 0.0f;
#pragma unroll
        for (int s4 = 0; s4 < KS / 4; ++s4) {
            uint4 kw[NT];
#pragma unroll
            for (int tile = 0; tile < NT; ++tile) kw[tile] = kb[C::k_at(8 * tile + g, 4 * s4 + t)];
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int tile = 0; tile < NT; ++tile) {
                    const uint32_t w = st == 0 ? kw[tile].x : st == 1 ? kw[tile].y : st == 2 ? kw[tile].z : kw[tile].w;
                    const uint32_t (&qq)[2 * RR] = qa[4 * s4 + st];
                    uint32_t b0, b1;
                    halves4<KIND>(w, b0, b1);
                    if (ROWS == 8)
                        mma16816(s[tile], qq[0], qq[0], qq[1], qq[1], b0, b1);
                    else
                        mma16816(s[tile], qq[0], qq[RR - 1], qq[RR], qq[2 * RR - 1], b0, b1);
                }
        }
        const bool masked = pos < first || pos + CK > min(first_end, last_end) || ok != (1u << GR) - 1u;
#pragma unroll
        for (int tile = 0; tile < NT; ++tile)
#pragma unroll
            for (int e = 0; e < 2 * RR; ++e) s[tile][e] *= ks[tile / 2];
        if (masked) {
#pragma unroll
            for (int tile = 0; tile < NT; ++tile)
#pragma unroll
                for (int e = 0; e < 2 * RR; ++e) {
                    const int key = pos + 8 * tile + 2 * t + (e & 1);
                    if (key < first || key >= end[e >> 1] || !((ok >> (tile / 2)) & 1u)) s[tile][e] = -INFINITY;
                }
        }
        float ms[RR];
        bool grew = false;
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) {
            float top = s[0][2 * rr];
#pragma unroll
            for (int tile = 0; tile < NT; ++tile) top = fmaxf(top, fmaxf(s[tile][2 * rr], s[tile][2 * rr + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            ms[rr] = fmaxf(m[rr], top);
            grew |= ms[rr] > m[rr];
        }
        float vmax = vs[0];
#pragma unroll
        for (int gi = 1; gi < GR; ++gi) vmax = fmaxf(vmax, vs[gi]);
        if (__any_sync(0xFFFFFFFFu, grew) || vmax > S) {
            const float Sn = fmaxf(S, vmax), fs = Sn > 0.0f ? S / Sn : 0.0f;
            float f[RR];
#pragma unroll
            for (int rr = 0; rr < RR; ++rr) {
                f[rr] = ms[rr] > -INFINITY ? ex2(m[rr] - ms[rr]) : 0.0f;
                l[rr] *= f[rr];
                m[rr] = ms[rr];
            }
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] *= f[RR == 1 ? 0 : e >> 1] * fs;
            S = Sn;
            invS = Sn > 0.0f ? 1.0f / Sn : 0.0f;
        }
        float mm[RR];
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) mm[rr] = m[rr] > -INFINITY ? m[rr] : 0.0f;
#pragma unroll
        for (int gi = 0; gi < GR; ++gi) {
            const float w = vs[gi] * invS;
            uint32_t ph[2 * RR], pl[2 * RR];  // [tile of the granule * RR + rr]
#pragma unroll
            for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                for (int rr = 0; rr < RR; ++rr) {
                    float p0 = ex2(s[2 * gi + tile][2 * rr] - mm[rr]), p1 = ex2(s[2 * gi + tile][2 * rr + 1] - mm[rr]);
                    l[rr] += p0 + p1;
                    p0 *= w;
                    p1 *= w;
                    float l0, l1;
                    ph[tile * RR + rr] = pack_hi(p0, p1, l0, l1);
                    pl[tile * RR + rr] = pack(l0, l1);
                }
            uint32_t vw[4][D / 32];  // D / 8 dims of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the granule
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int row = 16 * gi + 2 * t + (y & 1) + (y >> 1) * 8;
                if (D == 64) {
                    const uint2 z = reinterpret_cast<const uint2 *>(vb + C::v_at(row, g >> 1))[g & 1];
                    vw[y][0] = z.x;
                    vw[y][1] = z.y;
                } else {
                    const uint4 z = vb[C::v_at(row, g)];
                    vw[y][0] = z.x;
                    vw[y][1] = z.y;
                    vw[y][D / 32 - 2] = z.z;
                    vw[y][D / 32 - 1] = z.w;
                }
                // A granule that was not loaded holds what the ring held before, and a code behind the last
                // key may be NaN in e4m3: 0 * NaN is not 0.
                if (KIND == GPT2_KV8_E4M3 && masked && (pos + row >= n || !((ok >> gi) & 1u)))
#pragma unroll
                    for (int q = 0; q < D / 32; ++q) vw[y][q] = 0;
            }
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {  // 4 dims: column tiles 4 q .. 4 q + 3
                const uint32_t wk[4] = {vw[0][q], vw[1][q], vw[2][q], vw[3][q]};
                uint32_t b0[4], b1[4];
                pairs4<KIND>(wk[0], wk[1], b0);
                pairs4<KIND>(wk[2], wk[3], b1);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (ROWS == 8) {
                        mma16816(o[4 * q + j], ph[0], pl[0], ph[RR], pl[RR], b0[j], b1[j]);
                    } else {
                        mma16816(o[4 * q + j], ph[0], ph[RR - 1], ph[RR], ph[2 * RR - 1], b0[j], b1[j]);
                        mma16816(o[4 * q + j], pl[0], pl[RR - 1], pl[RR], pl[2 * RR - 1], b0[j], b1[j]);
                    }
                }
            }
        }
    };

    const int mine = chunks > warp ? (chunks - warp + NW - 1) / NW : 0;  // chunks warp, warp + NW, ...
    // The look-up of a set must come before the loads of its chunks but after the last use of the set before: scales
    // and validity of the chunks in flight are kept in registers, two sets deep.
    float pks[2] = {}, pvs[2] = {};  // this lane's granule scales of the even and odd set
    unsigned pok[2] = {};
    auto fetch = [&](int i) {
        if (i < mine) {
            if (i % SET == 0) {
                look_up(i / SET);
                const int b = (i / SET) & 1;
                if (b) pks[1] = gks, pvs[1] = gvs, pok[1] = gok;
                else pks[0] = gks, pvs[0] = gvs, pok[0] = gok;
            }
            load(i, i % STAGES);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();  // every lane's copies of chunk i are there, and all are done with chunk i - 1
        fetch(i + STAGES - 1);
        const bool odd = (i / SET) & 1;
        float ks[GR], vs[GR];
#pragma unroll
        for (int gi = 0; gi < GR; ++gi) {
            ks[gi] = __shfl_sync(0xFFFFFFFFu, odd ? pks[1] : pks[0], (i % SET) * GR + gi);
            vs[gi] = __shfl_sync(0xFFFFFFFFu, odd ? pvs[1] : pvs[0], (i % SET) * GR + gi);
        }
        const unsigned ok = ((odd ? pok[1] : pok[0]) >> ((i % SET) * GR)) & ((1u << GR) - 1u);
        compute(ring + i % STAGES * CHUNK_BYTES, lo + (i * NW + warp) * CK, ks, vs, ok);
    }
    if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(c.status, ST_KV8_BAD_PAGE);

    __syncthreads();  // every warp is through its ring
    // the warps' rows: thread (g, t) holds dims 16 t .. (D 64: columns j of tiles 2 t and 2 t + 1)
#pragma unroll
    for (int rr = 0; rr < RR; ++rr) {
        l[rr] += __shfl_xor_sync(0xFFFFFFFFu, l[rr], 1);
        l[rr] += __shfl_xor_sync(0xFFFFFFFFu, l[rr], 2);
        if (t == 0) {
            sm[warp][g + 8 * rr] = m[rr];
            sl[warp][g + 8 * rr] = l[rr];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < DT; j += 4) {
                float4 w;
                float *wf = reinterpret_cast<float *>(&w);
#pragma unroll
                for (int k = 0; k < 4; ++k) wf[k] = (RR == 1 ? o[j + k][e] + o[j + k][2 + e] : o[j + k][2 * rr + e]) * S;
                *reinterpret_cast<float4 *>(&so[warp][g + 8 * rr][(2 * t + e) * DT + j]) = w;
            }
    }
    __syncthreads();
    const int rows = min(ROWS, R - qt * ROWS);
    auto merged = [&](int row, int d, float &mx, float &lx) {
        mx = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row]));
        lx = 0.0f;
        float x = 0.0f;
        if (mx > -INFINITY) {
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = ex2(sm[w][row] - mx);
                lx = fmaf(f, sl[w][row], lx);
                x = fmaf(f, so[w][row][d], x);
            }
        }
        return x;
    };
    auto put = [&](int row, int d, float x) {
        const int i = qt * ROWS + row, tok = i / a.G;
        a.out[r * a.o_row + tok * a.o_tok + static_cast<long long>(h * a.G + (i - tok * a.G)) * D + d] = __float2half_rn(x);
    };
    if (active <= 1) {
        for (int e = threadIdx.x; e < rows * D; e += 32 * NW) {
            float mx, lx;
            const float x = merged(e / D, e % D, mx, lx);
            put(e / D, e % D, lx > 0.0f ? x / lx : 0.0f);
        }
        return;
    }
    const int tile = blockIdx.x / a.nsplit;
    const int prow = min(ROWS, R);  // rows of a tile in the work area
    float *part = a.part + static_cast<long long>(blockIdx.x - split) * prow * (D + 2);
    for (int e = threadIdx.x; e < rows * D; e += 32 * NW) {
        float mx, lx;
        const float x = merged(e / D, e % D, mx, lx);
        float *pr = part + (static_cast<long long>(split) * prow + e / D) * (D + 2);
        pr[e % D] = x;
        if (e % D == 0) {
            pr[D] = mx;
            pr[D + 1] = lx;
        }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned seen = atomicAdd(&a.arrive[tile], 1u);
        is_last = seen == static_cast<unsigned>(active - 1);
        if (is_last) a.arrive[tile] = 0;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    for (int e = threadIdx.x; e < rows * D; e += 32 * NW) {
        const float *pr = part + (e / D) * (D + 2);
        const long long step = static_cast<long long>(prow) * (D + 2);
        float mx = -INFINITY;
        for (int s = 0; s < active; ++s) mx = fmaxf(mx, __ldcg(pr + s * step + D));
        float lx = 0.0f, x = 0.0f;
        if (mx > -INFINITY)
#pragma unroll 4
            for (int s = 0; s < active; ++s) {
                const float f = ex2(__ldcg(pr + s * step + D) - mx);
                lx = fmaf(f, __ldcg(pr + s * step + D + 1), lx);
                x = fmaf(f, __ldcg(pr + s * step + e % D), x);
            }
        put(e / D, e % D, lx > 0.0f ? x / lx : 0.0f);
    }
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
    const kv8::Work w = kv8::work_layout(kv, Hq, Tq);
    if (!kv8::aligned(out) || !kv8::aligned(q) || (out_row_stride & 7) || (out_tok_stride & 7) || (q_row_stride & 7) ||
        (q_tok_stride & 7) || kv->work_bytes < w.bytes)
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    kv8::AttParams a;
    a.q = q;
    a.out = out;
    a.q_row = q_row_stride;
    a.q_tok = q_tok_stride;
    a.o_row = out_row_stride;
    a.o_tok = out_tok_stride;
    a.d_first = d_first;
    a.d_count = d_count;
    a.L = L;
    a.G = Hq / kv->nHead;
    a.Tq = Tq;
    a.count = count;
    a.max_len = max_len ? max_len : kv->maxPages * kv->page;
    a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(kv->headDim));
    const long long run = static_cast<long long>(kv->page) * kv->headDim;
    a.page_stride = run * kv->nHead * 2 * kv->nLayer;
    a.k_off = run * kv->nHead * 2 * L;
    a.v_off = a.k_off + run * kv->nHead;
    a.part = w.part;
    a.arrive = w.arrive;
    // Plan: whole (row, head, tile) units while they fill the GPU; else spans of at least NW chunks, about
    // WAVES CTAs per resident slot.
    const long long R = static_cast<long long>(a.G) * Tq;
    const int rows = R <= 8 ? 8 : 16;
    a.qtiles = static_cast<int>((R + rows - 1) / rows);
    const long long units = static_cast<long long>(kv->nRow) * kv->nHead * a.qtiles;
    const int chunk = kv8::NW * (2048 / kv->headDim);
    const int longest = a.max_len + 2048 / kv->headDim;  // `first` may start inside a chunk
    const long long target = std::min<long long>(static_cast<long long>(ctx->num_sms) * 6, kv8::MAX_SPLIT_CTAS);
    long long nsplit = std::max<long long>(1, target / units);
    nsplit = std::min<long long>(nsplit, (longest + chunk - 1) / chunk);
    a.span = static_cast<int>((longest + nsplit - 1) / nsplit + chunk - 1) / chunk * chunk;
    a.nsplit = (longest + a.span - 1) / a.span;
    if (units * a.nsplit > 0x7FFFFFFFll) return GPT2_B200_EINVAL;
    const kv8::View c = kv8::view(kv, ctx->status);
    bool *attr_done = &ctx->kv8_attr_done[(kv->kind == GPT2_KV8_INT8 ? 0 : 4) + (kv->headDim == 64 ? 0 : 2) + (rows == 8 ? 0 : 1)];
    auto go = [&](auto kern) {
        if (!*attr_done) {
            RelaxedCapture relaxed;
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kv8::RING_BYTES) != cudaSuccess)
                return GPT2_B200_ECUDA;
            *attr_done = true;
        }
        kern<<<static_cast<unsigned>(units * a.nsplit), 32 * kv8::NW, kv8::RING_BYTES, stream>>>(c, a);
        return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
    };
    if (kv->kind == GPT2_KV8_INT8) {
        if (kv->headDim == 64)
            return rows == 8 ? go(kv8::k_kv8_attend<GPT2_KV8_INT8, 64, 8>) : go(kv8::k_kv8_attend<GPT2_KV8_INT8, 64, 16>);
        return rows == 8 ? go(kv8::k_kv8_attend<GPT2_KV8_INT8, 128, 8>) : go(kv8::k_kv8_attend<GPT2_KV8_INT8, 128, 16>);
    }
    if (kv->headDim == 64)
        return rows == 8 ? go(kv8::k_kv8_attend<GPT2_KV8_E4M3, 64, 8>) : go(kv8::k_kv8_attend<GPT2_KV8_E4M3, 64, 16>);
    return rows == 8 ? go(kv8::k_kv8_attend<GPT2_KV8_E4M3, 128, 8>) : go(kv8::k_kv8_attend<GPT2_KV8_E4M3, 128, 16>);
}
