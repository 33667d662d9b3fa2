// kv8_attend.cu — attention over the paged 8-bit cache.
//
// out = softmax(q K^T / sqrt(D)) V with K = code * scale per block of keys: the scale is constant over a
// block, so it multiplies a key's score (K) and its probability (V), never the D elements. Online
// softmax in base 2: m, l and o are rescaled by 2^(m_old - m_new) when a row's maximum grows.
//
// A decode step reads 2 D + 8 / block bytes per key and K/V head once and does 4 D flops per key and query:
// HBM-bound, if the codes get into the tensor cores cheaply. So:
//   - the products are mma.m16n8k16 in fp16 with fp32 sums. A code is exact in fp16 and so is q; p * vscale is not,
//     and goes in as hi + lo (two fp16): rounding it to one fp16 alone would add an error of the size of the
//     output's own rounding. hi + lo keep 22 bits, or 2^-34 of the row's largest where that is more (see e below). With at
//     most 8 query rows (the decode step) the MMA's rows 8..15 are free and take lo; with 9 to 16 rows lo is a second MMA.
//     mma.sync's rate is far above what HBM feeds (64 MMAs of 8 cycles per 8 KB of codes).
//   - a warp takes CK keys at a time (64 for D 64, 32 for D 128: 8 KB of K and V) through a ring of its own in shared
//     memory (cp.async, the next chunk in flight while one is computed, no CTA barrier). The sum over dims (QK) may run in any
//     order of dims, so a thread's 16 neighbouring code bytes of one key are its operands for 4 k-steps; PV's sum over keys and its
//     column order are as free, so a thread reads 8 or 16 neighbouring dims of the 4 keys whose p it holds, and ends with
//     16 neighbouring output dims. The 16-byte granules of a chunk are permuted so that neither read has bank conflicts.
//   - a lane looks up the page and the two scales of one 16-key granule for the warp, 32 granules at a time, and
//     shuffles hand them out.
//   - p * vscale has fp16's range neither where scales are small nor where the keys with large p have small values and the others
//     count for the output. So p * vscale * 2^(PV_BITS - e) goes in, e following the row's largest log2(p * vscale) as m follows the
//     largest score, and o is kept in those units: an attention sink of small values, or a block of huge values that nobody
//     attends, costs the other keys nothing.
//   - m is not the maximum but within 2^LAZY of it: p stays below 2^LAZY, far inside fp32, and most chunks need neither the row
//     maximum's shuffles nor a rescaling of o. So with e: p * vscale goes in at up to 2^(LAZY + PV_BITS) = 2^15.
//
// Work: a unit is (cache row, tile of 8 or 16 query rows, K/V head) with its chunks of keys, which the warps of a CTA (1, 2 or 4)
// take in turn; at its end they are merged in shared memory. With units in plenty each has a CTA. With fewer units than resident
// CTAs all chunks of all units form one sequence and every CTA takes an equal piece of it, found from the rows' lengths by a
// prefix sum, its loads running ahead over unit borders; a unit cut by a piece's end is merged through the work area by the last
// CTA to arrive, in piece order.
//
// Beams share their leading pages, and one query row of each fills an eighth of an MMA tile. With units in plenty and at most 4
// query rows in each, a CTA so takes 2 or 4 neighbouring cache rows of a head (GROUP). It compares their table rows; the chunks
// of the pages that all of them hold are read and converted once, for the query rows of all. The rows' own chunks follow, in
// which the other rows' scores are masked. 32 items x 4 beams x 12 heads of 640 to 700 keys, 640 shared: 14.4 us, each row by
// itself 29.0. Rows that share nothing gain a little from four warps to deal their chunks to (128 x 12 heads of 2048 to 4096 keys:
// 128 us, by themselves 146).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "ptx.cuh"

namespace b200 {
namespace kv8 {

constexpr int NW_PIECES = 4;         // warps per CTA of a launch in equal pieces, and of a group
constexpr float LAZY = 6.0f;         // log2 of how far a row's scores may pass m before m follows, and its p * vscale e
constexpr float PV_BITS = 9.0f;      // log2 of what the row's largest p * vscale goes in as
// Scores are not rounded before m is subtracted (one FMA), m is: beyond 2^28 that alone could be more than fp32's exponents. From
// STEEP on, where it is still 2^-8, scores are rounded as m is, and m and e follow every chunk.
constexpr float STEEP = 65536.0f;
constexpr float E_LEAST = -100.0f;   // e's least: what is below that is 0 in any fp16 output
constexpr int MAX_ENTRIES = 1024;    // (row, tile) pairs of a launch whose CTAs take equal pieces
constexpr int MAX_PIECES = 1024;     // CTAs of such a launch

int attend_max_ctas() { return 2 * MAX_PIECES; }  // a piece cuts two units at most

struct AttParams {
    const __half *q;
    __half *out;
    long long q_row, q_tok, o_row, o_tok;
    const int *d_first, *d_count;
    unsigned page_runs, k_run;  // runs of a page (layers x 2 x heads), of it before this layer's K
    float *part;
    unsigned *arrive;
    int L, G, Tq, count, max_len;
    int qtiles, entries;  // entries: (row, tile) pairs of a launch in equal pieces, 0: one unit per CTA
    float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with a zero accumulator.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// A copy that the compiler takes for another value. An MMA's four A operands are neighbouring registers: a value
// that is two of them would be moved there before every MMA.
__device__ __forceinline__ uint32_t twin(uint32_t v) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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

// A warp's chunk of CK keys in shared memory: K rows, then V rows, half of it each, in 16-byte granules.
// Reads: K, a quarter warp takes granules 0..3 (then 4..7 for D 128) of two neighbouring rows; V, a half warp takes two
// granules (8 bytes a lane) or a quarter warp two granules (16 bytes a lane) of rows 0, 2, 4, 6 of an 8-row
// group. The maps put each such set on 8 different bank groups (granule index mod 8).
constexpr int CHUNK_BYTES = 8192, HALF = CHUNK_BYTES / 2;
template <int D>
struct Chunk {
    static constexpr int CK = CHUNK_BYTES / 2 / D, GR = CK / 16, ROWG = D / 16;  // granules per row
    __device__ static int k_at(int row, int gr) { return row * ROWG + (D == 64 ? gr : gr ^ ((row & 1) << 2)); }
    __device__ static int v_at(int row, int gr) {
        if (D == 64) {  // 8-row groups: row bits (b2 b1 b0) stored as (b2 b0 b1); the granule's high bit flipped by b2
            const int at = (row & ~3) | ((row & 1) << 1) | ((row >> 1) & 1);
            return at * ROWG + (gr ^ ((row >> 1) & 2));
        }
        return row * ROWG + (gr ^ (row & 6));
    }
};

// A kernel variant's shape: 12 warps per SM, each with two chunks in its ring (192 KB of an SM's shared memory). The accumulators
// of 128 dims or 16 rows take the registers, so q of 128 dims lies in shared memory instead (32 registers), and the warps'
// rows are merged where the rings were or, in the middle of a piece, DH dims at a time in q's place.
// 16 rows of 128 dims spill at 12 warps, so 8 (8 sequences x 8 heads of 16384 keys: 62.5 us, 12 warps 68.7; 55.5 since the merge
// takes four dims per thread and the last CTA has the loads of all its rows in flight, 55.8 with e).
template <int D, int ROWS, int NW>
struct Shape {
    static constexpr int WARPS = D == 128 && ROWS == 16 ? 8 : 12;  // per SM
    static constexpr int RESIDENT = WARPS / NW;
    static constexpr int STAGES = 2;
    static constexpr int RING = NW * STAGES * CHUNK_BYTES;
    static constexpr int DH = 512 / ROWS, LOG_D = D == 64 ? 6 : 7, LOG_DH = ROWS == 8 ? 6 : 5;  // dims merged at a time
    static constexpr int SO = NW * ROWS * (DH + 4) * 4;
    static constexpr bool Q_SMEM = D == 128;
    static constexpr int QS = Q_SMEM ? D / 16 * 512 : 0;
    static constexpr int BYTES = RING + (SO > QS ? SO : QS);
    static_assert(NW == 1 || RESIDENT * (BYTES + 1024 + 160 * NW) <= 228 * 1024, "shared memory, with the CTA's 1 KB and the static arrays");
};

// GROUP: 0, or the cache rows of a CTA that reads their shared pages once (2 or 4)
template <int KIND, int D, int ROWS, int NW, int GROUP>
__global__ void __launch_bounds__(32 * NW, Shape<D, ROWS, NW>::RESIDENT) k_kv8_attend(const View c, const AttParams a) {
    using C = Chunk<D>;
    using SH = Shape<D, ROWS, NW>;
    constexpr int STAGES = SH::STAGES, RING_BYTES = SH::RING, DH = SH::DH;
    constexpr int CK = C::CK, GR = C::GR, NT = CK / 8, KS = D / 16, DT = D / 8, RR = ROWS / 8;
    constexpr int SET = 32 / GR;  // chunks whose granules one look-up covers
    extern __shared__ __align__(128) uint8_t ring_all[];
    uint4 *qs = reinterpret_cast<uint4 *>(ring_all + RING_BYTES);  // [KS][32]: A operands of a k-step
    int *pre = reinterpret_cast<int *>(ring_all + SH::BYTES);               // [entries + 1]: chunks before each entry
    __shared__ float sm[NW][ROWS], sl[NW][ROWS];
    __shared__ int is_last, warp_sum[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int R = a.G * a.Tq;
    const bool one = a.Tq == 1;  // then no row needs a division to find its token

    // Entry e: row r, its tile qt, the keys [first, last_end) that some query of the tile sees, in chunks from base on.
    int r, qt, n, first, base, last_end;
    auto entry = [&](int e) {
        r = e, qt = 0;
        if (a.qtiles > 1) {
            r = e / a.qtiles;
            qt = e - r * a.qtiles;
        }
        n = c.len[r] + (a.d_count ? a.d_count[r] : a.count);
        if (n < 0 || n > a.max_len) n = -1;
        first = a.d_first ? max(a.d_first[r], 0) : 0;
        last_end = one ? n : n - a.Tq + (min(qt * ROWS + ROWS, R) - 1) / a.G + 1;
        base = first & ~(CK - 1);
        return last_end > first ? (last_end - base + CK - 1) / CK : 0;
    };
    auto put = [&](int h, int row, int d, float4 y) {  // dims d .. d + 3
        int i = qt * ROWS + row, r_ = r;
        if (GROUP) {
            const int u = row / R;
            r_ = GROUP * blockIdx.x + u;
            i = row - u * R;
        }
        const int tok = one ? 0 : i / a.G;
        __half2 v[2] = {__floats2half2_rn(y.x, y.y), __floats2half2_rn(y.z, y.w)};
        *reinterpret_cast<uint2 *>(&a.out[r_ * a.o_row + tok * a.o_tok + static_cast<long long>(h * a.G + (i - tok * a.G)) * D + d]) =
            *reinterpret_cast<uint2 *>(v);
    };
    auto no_keys = [&](int h, int rows) {
        for (int x = 4 * tid; x < rows * D; x += 128 * NW) put(h, x / D, x % D, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    };

    // One unit per CTA: the pages of a warp's first granules, whatever the row's length, so that the table is read while the
    // length is.
    const bool early = !GROUP && !a.entries && !a.d_first && a.qtiles == 1;
    int early_page = -1;
    if (early) {
        const int pos = ((lane / GR) * NW + warp) * CK + (lane % GR) * 16;
        if (pos < a.max_len) early_page = c.table[static_cast<long long>(blockIdx.x) * c.maxPages + (pos >> c.page_shift)];
    }
    int c0, c1, per = 1;  // this CTA's chunks
    // A group's chunks: shared ones [0, first_of[0]) for all rows, then row i's own [first_of[i], first_of[i + 1]).
    __shared__ int first_of[GROUP + 1], len_of[GROUP + 1], differ;
    const int in_group = GROUP ? min(GROUP, c.nRow - GROUP * static_cast<int>(blockIdx.x)) : 1;
    if (GROUP) {
        const int r0 = GROUP * blockIdx.x;
        if (tid == 0) differ = 0x7FFFFFFF;
        if (tid < GROUP) {
            int x = tid < in_group ? c.len[r0 + tid] + (a.d_count ? a.d_count[r0 + tid] : a.count) : 0;
            if (x < 0 || x > a.max_len) {
                if (blockIdx.y == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
                x = 0;
            }
            len_of[tid] = x;
        }
        __syncthreads();
        int least = 0x7FFFFFFF;  // keys that every query of every row sees
        for (int i = 0; i < in_group; ++i) least = min(least, len_of[i] - a.Tq + 1);
        const int *t0 = c.table + static_cast<long long>(r0) * c.maxPages;
        const int pages = in_group > 1 && least > 0 ? ((least - 1) >> c.page_shift) + 1 : 0;
        for (int p = tid; p < pages; p += 32 * NW) {
            bool same = true;
            for (int i = 1; i < in_group; ++i) same &= t0[p] == t0[static_cast<long long>(i) * c.maxPages + p];
            if (!same) {
                atomicMin(&differ, p);
                break;
            }
        }
        __syncthreads();
        if (tid == 0) {
            int at = in_group > 1 ? max(0, differ < pages ? differ << c.page_shift : least) / CK : 0;
            const int from = at;
            for (int i = 0; i < GROUP; ++i) {
                first_of[i] = at;
                at += max(0, (len_of[i] + CK - 1) / CK - from);
            }
            first_of[GROUP] = at;
        }
        __syncthreads();
        r = r0, qt = 0, first = 0, base = 0;
        n = last_end = 0x7FFFFFFF;
        c0 = 0;
        c1 = first_of[GROUP];
        if (c1 == 0) no_keys(blockIdx.y, in_group * R);
    } else if (a.entries) {
        const int own = (a.entries + 32 * NW - 1) / (32 * NW), e0 = min(tid * own, a.entries), e1 = min(e0 + own, a.entries);
        int sum = 0;
        for (int e = e0; e < e1; ++e) {
            pre[e] = sum;
            const int ch = entry(e);
            sum += ch * c.nHead;
            if (n < 0 && blockIdx.x == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        }
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += u;
        }
        if (lane == 31) warp_sum[warp] = before;
        before -= sum;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += warp_sum[w];
            total += warp_sum[w];
        }
        for (int e = e0; e < e1; ++e) pre[e] += before;
        if (tid == 0) pre[a.entries] = total;
        __syncthreads();
        per = ((total + gridDim.x - 1) / gridDim.x + NW - 1) & ~(NW - 1);
        c0 = min(static_cast<long long>(blockIdx.x) * per, static_cast<long long>(total));
        c1 = min(c0 + per, total);
        for (int e = blockIdx.x; e < a.entries; e += gridDim.x)
            if (pre[e] == pre[e + 1]) {
                entry(e);
                for (int h = 0; h < c.nHead; ++h) no_keys(h, min(ROWS, R - qt * ROWS));
            }
    } else {
        c0 = 0;
        c1 = entry(blockIdx.x);
        if (n < 0 && tid == 0 && blockIdx.y == 0) atomicOr(c.status, ST_KV8_BAD_LEN);
        if (c1 == 0) no_keys(blockIdx.y, min(ROWS, R - qt * ROWS));
    }
    // The unit of chunk x: sets entry()'s values, h and the unit's first chunk u0; returns its chunks.
    int h = blockIdx.y, u0 = 0;
    auto unit_of = [&](int x) {
        if (GROUP) return c1;
        int e = blockIdx.x;
        if (a.entries) {
            int lo = 0, hi = a.entries;  // the last entry with pre <= x (entries without chunks come before it)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pre[mid] <= x) lo = mid;
                else hi = mid;
            }
            e = lo;
        }
        const int ch = entry(e);
        if (a.entries) {
            h = (x - pre[e]) / ch;
            u0 = pre[e] + h * ch;
        }
        return ch;
    };

    // GROUP: the row whose own chunk x is (-1: a shared one), and its first key.
    auto chunk_of = [&](int x, int &key) {
        int i = -1;
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
            if (x >= first_of[u] && x < first_of[u + 1]) i = u;
        key = (i < 0 ? x : x - first_of[i] + first_of[0]) * CK;
        return i;
    };
    // This lane's granule of the set looked up last: its first code row of K (rows are counted in 32 bits) and its scales, which
    // nothing waits for before the set's first chunk is computed.
    unsigned grow = 0;
    float gks = 0.0f, gvs = 0.0f;
    unsigned gok = 0;
    // A block of zeros has scale 0; TINY in its place keeps -inf (a masked score) times a scale from being NaN.
    constexpr float TINY = 1e-20f;
    bool bad = false;
    auto look_up = [&](int set) {
        const int r_ = r, qt_ = qt, n_ = n, first_ = first, base_ = base, last_end_ = last_end, h_ = h, u0_ = u0;
        const int x = c0 + (set * SET + lane / GR) * NW + warp;
        int ok = x < c1, pos = 0;
        if (GROUP) {
            if (ok) {
                const int own = chunk_of(x, pos);
                pos += (lane % GR) * 16;
                ok = own < 0 || pos < len_of[own];
                r = GROUP * blockIdx.x + max(own, 0);
            }
        } else if (ok) {
            unit_of(x);
            pos = base + (x - u0) * CK + (lane % GR) * 16;
            ok = pos < last_end && pos + 16 > first;
        }
        if (ok) {
            const int p = early && set == 0 ? early_page : c.table[static_cast<long long>(r) * c.maxPages + (pos >> c.page_shift)];
            if (p < 0 || p >= c.nPages) {
                bad = true;
                ok = 0;
            } else {
                const unsigned ip = pos & (c.page - 1), run = p * a.page_runs + a.k_run + h;
                const int sub = c.page_shift - c.block_shift;
                gks = c.scale[(run << sub) + (ip >> c.block_shift)];
                gvs = c.scale[((run + c.nHead) << sub) + (ip >> c.block_shift)];
                grow = (run << c.page_shift) + ip;
            }
        }
        if (!ok) gks = gvs = 0.0f;
        gok = __ballot_sync(0xFFFFFFFFu, ok);
        r = r_, qt = qt_, n = n_, first = first_, base = base_, last_end = last_end_, h = h_, u0 = u0_;
    };
    uint8_t *ring = ring_all + warp * STAGES * CHUNK_BYTES;
    const uint32_t ring_s = smem_u32(ring);
    // A copy instruction of the warp takes 512 bytes: 8 rows (D 64) or 4. V's rows are dealt to the lanes so that its
    // stores, too, meet 8 bank groups per 8 lanes.
    const int krow = lane / C::ROWG;
    const int vrow = D == 64 ? ((lane >> 2) & 1) * 2 + ((lane >> 3) & 1) + (lane >> 4) * 4 : krow;
    const int cgr = lane & (C::ROWG - 1);
    constexpr int CR = 32 / C::ROWG;  // rows per copy instruction
    const uint8_t *kbase = c.data + krow * D + cgr * 16;
    const uint8_t *vbase = c.data + vrow * D + cgr * 16 + (static_cast<size_t>(c.nHead) << c.page_shift) * D;
    // C::k_at and C::v_at of this lane's granule, without the multiples of 8 (D 64) or 4 rows that are immediates below
    const int ko = C::k_at(krow, cgr) * 16, vo0 = HALF + C::v_at(vrow, cgr) * 16, vo1 = HALF + C::v_at(vrow, cgr ^ (D == 64 ? 0 : 4)) * 16;
    auto load = [&](int i, int stage) {  // chunk i of this warp; its set has been looked up
        const uint32_t dst = ring_s + stage * CHUNK_BYTES;
#pragma unroll
        for (int gi = 0; gi < GR; ++gi) {
            const int src_lane = (i % SET) * GR + gi;
            const unsigned row0 = __shfl_sync(0xFFFFFFFFu, grow, src_lane);
            if (!((gok >> src_lane) & 1u)) continue;
            const uint8_t *kp = kbase + static_cast<size_t>(row0) * D, *vp = vbase + static_cast<size_t>(row0) * D;
#pragma unroll
            for (int x = 0; x < 16 / CR; ++x) {
                const int at = (gi * 16 + x * CR) * D;
                cp_async16(dst + ko + at, kp + x * CR * D);
                cp_async16(dst + (x & 1 ? vo1 : vo0) + at, vp + x * CR * D);
            }
        }
    };
    // Shared-memory offsets of this lane's reads, so that all but an immediate is computed once (C::k_at, C::v_at).
    const int kl0 = (D == 64 ? g * 4 + t : g * 8 + (t ^ ((g & 1) << 2))) * 16;
    const int kl1 = D == 64 ? 0 : (g * 8 + ((4 + t) ^ ((g & 1) << 2))) * 16;
    const int vl = HALF + (D == 64 ? ((((t >> 1) * 4 + (t & 1)) * 4 + ((g >> 1) ^ (t & 2))) * 16 + (g & 1) * 8)
                                   : (2 * t * 8 + (g ^ (2 * t))) * 16);
    // The segment at hand: q, m, e, l, o and the keys its rows see.
    __align__(16) uint32_t qa[SH::Q_SMEM ? 1 : KS][4];  // A operands: with 8 rows, rows 8..15 are rows 0..7 again
    int my_row = 0;  // GROUP: the cache row, in the group, of this lane's query row
    int end[RR], full_end = 0;  // keys of every row: [first, full_end)
    float o[DT][4], m[RR], l[RR], e2[RR], pv[RR];  // e; 2^(PV_BITS - e)
    bool steep = false;  // some row's |m| is over STEEP
    auto compute = [&](const bool masked, const bool other, const uint8_t *buf, int pos, float (&ks)[GR], float (&vs)[GR], float most, unsigned ok) {
        float s[NT][4];
#pragma unroll
        for (int s4 = 0; s4 < KS / 4; ++s4) {
            uint4 kw[NT];
#pragma unroll
            for (int tile = 0; tile < NT; ++tile) kw[tile] = *reinterpret_cast<const uint4 *>(buf + (s4 ? kl1 : kl0) + tile * 8 * D);
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int tile = 0; tile < NT; ++tile) {
                    const uint32_t w = st == 0 ? kw[tile].x : st == 1 ? kw[tile].y : st == 2 ? kw[tile].z : kw[tile].w;
                    if (SH::Q_SMEM && tile == 0) *reinterpret_cast<uint4 *>(qa[0]) = qs[(4 * s4 + st) * 32 + lane];
                    const uint32_t (&qq)[4] = qa[SH::Q_SMEM ? 0 : 4 * s4 + st];
                    uint32_t b0, b1;
                    halves4<KIND>(w, b0, b1);
                    if (s4 == 0 && st == 0) mma16816_first(s[tile], qq[0], qq[1], qq[2], qq[3], b0, b1);
                    else mma16816(s[tile], qq[0], qq[1], qq[2], qq[3], b0, b1);
                }
        }
        if (masked) {
#pragma unroll
            for (int tile = 0; tile < NT; ++tile)
#pragma unroll
                for (int e = 0; e < 2 * RR; ++e) {
                    const int key = pos + 8 * tile + 2 * t + (e & 1);
                    if (key < first || key >= end[e >> 1] || !((ok >> (tile / 2)) & 1u)) s[tile][e] = -INFINITY;
                }
        }
        if (GROUP && other)
#pragma unroll
            for (int tile = 0; tile < NT; ++tile) s[tile][0] = s[tile][1] = -INFINITY;
        // A granule's scale is one factor of its scores: the largest of them first, then the factor.
        auto largest = [&](int rr, int gi) {
            return ks[gi] * fmaxf(fmaxf(s[2 * gi][2 * rr], s[2 * gi][2 * rr + 1]), fmaxf(s[2 * gi + 1][2 * rr], s[2 * gi + 1][2 * rr + 1]));
        };
        float top[RR];
        bool grew = steep;
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) {
            top[rr] = -INFINITY;
#pragma unroll
            for (int gi = 0; gi < GR; ++gi) top[rr] = fmaxf(top[rr], largest(rr, gi));
            // m -inf: any key. most, the chunk's largest log2(vscale), stands for every granule's: e is looked at closer below
            grew |= top[rr] + fmaxf(most - e2[rr], 0.0f) > m[rr] + LAZY;
        }
        if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
            for (int rr = 0; rr < RR; ++rr) {
                top[rr] = fmaxf(top[rr], __shfl_xor_sync(0xFFFFFFFFu, top[rr], 1));
                top[rr] = fmaxf(top[rr], __shfl_xor_sync(0xFFFFFFFFu, top[rr], 2));
                const float mn = fmaxf(m[rr], top[rr]), fell = m[rr] - mn;  // NaN as long as there is no key
                const bool some = mn > -INFINITY;
                float en = -INFINITY;
#pragma unroll
                for (int gi = 0; gi < GR; ++gi) en = fmaxf(en, (largest(rr, gi) - mn) + lg2(vs[gi]));
                en = fmaxf(en, __shfl_xor_sync(0xFFFFFFFFu, en, 1));
                en = fmaxf(en, __shfl_xor_sync(0xFFFFFFFFu, en, 2));
                en = fmaxf(fmaxf(en, e2[rr] + fell), E_LEAST);
                const float f = some ? ex2((e2[rr] + fell) - en) : 0.0f;
                m[rr] = mn;
                e2[rr] = en;
                pv[rr] = ex2(PV_BITS - en);
                l[rr] *= some ? ex2(fell) : 0.0f;
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    o[j][RR == 1 ? 0 : 2 * rr] *= f;
                    o[j][RR == 1 ? 1 : 2 * rr + 1] *= f;
                    if (RR == 1) {
                        o[j][2] *= f;
                        o[j][3] *= f;
                    }
                }
            }
            bool far = false;
#pragma unroll
            for (int rr = 0; rr < RR; ++rr) far |= fabsf(m[rr]) > STEEP && fabsf(m[rr]) < INFINITY;
            steep = __any_sync(0xFFFFFFFFu, far);
            if (steep) {  // round the scores as the maximum was
#pragma unroll
                for (int gi = 0; gi < GR; ++gi) {
#pragma unroll
                    for (int e = 0; e < 2 * RR; ++e) {
                        s[2 * gi][e] *= ks[gi];
                        s[2 * gi + 1][e] *= ks[gi];
                    }
                    ks[gi] = 1.0f;
                }
            }
        }
        float mm[RR];
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) mm[rr] = m[rr] > -INFINITY ? m[rr] : 0.0f;
#pragma unroll
        for (int gi = 0; gi < GR; ++gi) {
            uint32_t ph[2 * RR], pl[2 * RR];  // [tile of the granule * RR + rr]
#pragma unroll
            for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                for (int rr = 0; rr < RR; ++rr) {
                    float p0 = ex2(fmaf(s[2 * gi + tile][2 * rr], ks[gi], -mm[rr]));
                    float p1 = ex2(fmaf(s[2 * gi + tile][2 * rr + 1], ks[gi], -mm[rr]));
                    l[rr] += p0 + p1;
                    const float w = other ? 0.0f : vs[gi] * pv[rr];
                    p0 *= w;
                    p1 *= w;
                    float l0, l1;
                    ph[tile * RR + rr] = pack_hi(p0, p1, l0, l1);
                    pl[tile * RR + rr] = pack(l0, l1);
                }
            uint32_t vw[4][D / 32];  // D / 8 dims of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the granule
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint8_t *vp = buf + vl + (D == 64 ? 16 * gi + 8 * (y >> 1) + 2 * (y & 1) : 16 * gi + 8 * (y >> 1) + (y & 1)) * D;
                if (D == 64) {
                    const uint2 z = *reinterpret_cast<const uint2 *>(vp);
                    vw[y][0] = z.x;
                    vw[y][1] = z.y;
                } else {
                    const uint4 z = *reinterpret_cast<const uint4 *>(vp);
                    vw[y][0] = z.x;
                    vw[y][1] = z.y;
                    vw[y][D / 32 - 2] = z.z;
                    vw[y][D / 32 - 1] = z.w;
                }
            }
            // A granule that was not loaded holds what the ring held before, and a code behind the last
            // key may be NaN in e4m3: 0 * NaN is not 0.
            if (KIND == GPT2_KV8_E4M3 && masked)
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    if (pos + 16 * gi + 2 * t + (y & 1) + (y >> 1) * 8 >= n || !((ok >> gi) & 1u))
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) vw[y][q] = 0;
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {  // 4 dims: column tiles 4 q .. 4 q + 3
                uint32_t b0[4], b1[4];
                pairs4<KIND>(vw[0][q], vw[1][q], b0);
                pairs4<KIND>(vw[2][q], vw[3][q], b1);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (ROWS == 8) mma16816(o[4 * q + j], ph[0], pl[0], ph[RR], pl[RR], b0[j], b1[j]);
                    else mma16816(o[4 * q + j], ph[0], ph[RR - 1], ph[RR], ph[2 * RR - 1], b0[j], b1[j]);
                }
                if (ROWS == 16)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma16816(o[4 * q + j], pl[0], pl[RR - 1], pl[RR], pl[2 * RR - 1], b0[j], b1[j]);
            }
        }
    };

    const int mine = c1 - c0 > warp ? (c1 - c0 - warp + NW - 1) / NW : 0;  // chunks c0 + warp, c0 + warp + NW, ...
    // The look-up of a set comes before the loads of its chunks, while the set before is still in use: pks, pvs and pok are
    // the set's in use, pmost the chunk's largest log2(vscale) in the lanes of its granules.
    float pks = TINY, pvs = 0.0f, pmost = -INFINITY;
    unsigned pok = 0;
    auto fetch = [&](int i) {
        if (i < mine) {
            if (i % SET == 0) look_up(i / SET);
            load(i, i % STAGES);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
    int i = 0;
    for (int x0 = c0; x0 < c1;) {
        const int u1 = unit_of(x0) + u0, x1 = min(u1, c1);
        full_end = one ? n : min(n - a.Tq + qt * ROWS / a.G + 1, last_end);
        // q: thread (g, t) holds dims 64 * (s / 4) + 16 t + 4 (s % 4) .. + 3 of row g (and g + 8) for k-step s
        if (SH::Q_SMEM) __syncthreads();  // every warp is through with the last segment's q
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) {
            int row = qt * ROWS + g + 8 * rr, cr = r, keys = n;
            bool ok = row < R;
            if (GROUP) {
                my_row = g / R;
                ok = my_row < in_group;
                row = g - my_row * R;
                cr = r + (ok ? my_row : 0);
                keys = ok ? len_of[my_row] : 0;
            }
            const int tok = ok && !one ? row / a.G : 0;
            end[rr] = ok ? keys - a.Tq + tok + 1 : 0;
            const __half *qp = a.q + cr * a.q_row + tok * a.q_tok + static_cast<long long>(h * a.G + (row - tok * a.G)) * D + 16 * t;
#pragma unroll
            for (int s4 = 0; s4 < KS / 4; ++s4) {
                if (SH::Q_SMEM && s4 % NW != warp) continue;  // the warps share the work
                uint4 x[2] = {};
                if (ok) {
                    x[0] = *reinterpret_cast<const uint4 *>(qp + 64 * s4);
                    x[1] = *reinterpret_cast<const uint4 *>(qp + 64 * s4 + 8);
                }
                const uint32_t *w = reinterpret_cast<const uint32_t *>(x);
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    if (SH::Q_SMEM) {
                        uint32_t *dst = reinterpret_cast<uint32_t *>(qs + (4 * s4 + s) * 32 + lane);
                        dst[rr] = w[2 * s];
                        dst[2 + rr] = w[2 * s + 1];
                        if (RR == 1) {
                            dst[1] = w[2 * s];
                            dst[3] = w[2 * s + 1];
                        }
                    } else {
                        uint32_t (&dst)[4] = qa[SH::Q_SMEM ? 0 : 4 * s4 + s];
                        dst[rr] = w[2 * s];
                        dst[2 + rr] = w[2 * s + 1];
                        if (RR == 1) {
                            dst[1] = twin(w[2 * s]);
                            dst[3] = twin(w[2 * s + 1]);
                        }
                    }
                }
            }
            m[rr] = -INFINITY;
            l[rr] = 0.0f;
            e2[rr] = E_LEAST;
            pv[rr] = 0.0f;
        }
        steep = false;
        if (SH::Q_SMEM) __syncthreads();
#pragma unroll
        for (int j = 0; j < DT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        for (; c0 + i * NW + warp < x1; ++i) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of chunk i are there, and all are done with chunk i - 1
            fetch(i + STAGES - 1);
            if (i % SET == 0) {
                pks = fmaxf(gks * a.scale_log2, TINY);
                pvs = gvs;
                pok = gok;
                pmost = gvs;
#pragma unroll
                for (int x = 1; x < GR; x <<= 1) pmost = fmaxf(pmost, __shfl_xor_sync(0xFFFFFFFFu, pmost, x));
                pmost = lg2(pmost);
            }
            float ks[GR], vs[GR];
#pragma unroll
            for (int gi = 0; gi < GR; ++gi) {
                ks[gi] = __shfl_sync(0xFFFFFFFFu, pks, (i % SET) * GR + gi);
                vs[gi] = __shfl_sync(0xFFFFFFFFu, pvs, (i % SET) * GR + gi);
            }
            const float most = __shfl_sync(0xFFFFFFFFu, pmost, (i % SET) * GR);
            const unsigned ok = (pok >> ((i % SET) * GR)) & ((1u << GR) - 1u);
            int pos = base + (c0 + i * NW + warp - u0) * CK;
            bool other = false;  // GROUP: a chunk of another row than this lane's
            if (GROUP) {
                const int own = chunk_of(i * NW + warp, pos);
                other = own >= 0 && own != my_row;
                n = own < 0 ? 0x7FFFFFFF : len_of[max(own, 0)];
                full_end = own < 0 ? 0x7FFFFFFF : n - a.Tq + 1;
            }
            const uint8_t *buf = ring + i % STAGES * CHUNK_BYTES;
            const bool masked = pos < first || pos + CK > full_end || ok != (1u << GR) - 1u;
            compute(masked, other, buf, pos, ks, vs, most, ok);
        }
        // The warps' rows: behind the last chunk all dims at a time, each warp's in its own ring; before, when the next unit's
        // chunks are there or on their way, DH dims at a time. Thread (g, t) holds dims 2 t DT .. (the columns j of tiles 2 t and
        // 2 t + 1).
        const bool idle = x1 == c1;
        const int dlog = idle ? SH::LOG_D : SH::LOG_DH, tlog = dlog - SH::LOG_D + 2;  // threads t of a part
        float *const merge = reinterpret_cast<float *>(idle ? ring_all : ring_all + RING_BYTES);
        const int row_step = (1 << dlog) + 4, warp_step = idle ? RING_BYTES / NW / 4 : ROWS * (DH + 4);
        const int rows = GROUP ? in_group * R : min(ROWS, R - qt * ROWS);
        constexpr bool PIECES = NW == NW_PIECES && !GROUP;
        const bool whole = !PIECES || (u0 >= c0 && u1 <= c1);
        const int prow = min(ROWS, R);  // rows of a tile in the work area
        const int slot = 2 * blockIdx.x + (x0 == c0 ? 0 : 1);
#pragma unroll
        for (int rr = 0; rr < RR; ++rr) {
            l[rr] += __shfl_xor_sync(0xFFFFFFFFu, l[rr], 1);
            l[rr] += __shfl_xor_sync(0xFFFFFFFFu, l[rr], 2);
            if (l[rr] != l[rr]) m[rr] = fmaxf(m[rr], 0.0f);  // NaN stays: a row without keys (m -inf) is left out of the merge
        }
#pragma unroll 1
        for (int part = 0; part < D >> dlog; ++part) {
            if (x0 > c0 || !idle) __syncthreads();  // the last merge is through, and all warps with q
            else __syncwarp();
            if (t >> tlog == part) {
                const int tp = t - (part << tlog);
#pragma unroll
                for (int rr = 0; rr < RR; ++rr) {
                    if (tp == 0) {
                        sm[warp][g + 8 * rr] = m[rr];
                        sl[warp][g + 8 * rr] = l[rr];
                    }
                    const float unit = ex2(e2[rr] - PV_BITS);
                    float *to = merge + warp * warp_step + (g + 8 * rr) * row_step + 2 * tp * DT;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < DT; j += 4) {
                            float4 w;
                            float *wf = reinterpret_cast<float *>(&w);
#pragma unroll
                            for (int k = 0; k < 4; ++k) wf[k] = (RR == 1 ? o[j + k][e] + o[j + k][2 + e] : o[j + k][2 * rr + e]) * unit;
                            *reinterpret_cast<float4 *>(to + e * DT + j) = w;
                        }
                }
            }
            __syncthreads();
            for (int x = tid; x < rows << (dlog - 2); x += 32 * NW) {
                const int row = x >> (dlog - 2), dh = 4 * (x - (row << (dlog - 2))), d = (part << dlog) + dh;
                float mx = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm[w][row]);
                float lx = 0.0f;
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (mx > -INFINITY) {
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const float f = ex2(sm[w][row] - mx);
                        const float4 z = *reinterpret_cast<const float4 *>(merge + w * warp_step + row * row_step + dh);
                        lx = fmaf(f, sl[w][row], lx);
                        y = make_float4(fmaf(f, z.x, y.x), fmaf(f, z.y, y.y), fmaf(f, z.z, y.z), fmaf(f, z.w, y.w));
                    }
                }
                if (whole) {
                    const float inv = lx != 0.0f ? 1.0f / lx : 0.0f;  // NaN stays NaN
                    put(h, row, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                } else {
                    float *pr = a.part + static_cast<long long>(slot) * prow * (D + 4);  // [prow][D] o, [prow][2] m, l, 16-byte steps
                    *reinterpret_cast<float4 *>(pr + row * D + d) = y;
                    if (d == 0) *reinterpret_cast<float2 *>(pr + prow * D + 2 * row) = make_float2(mx, lx);
                }
            }
        }
        if (PIECES && !whole) {  // pieces k0 .. k1 share the unit; its first piece's slot names its counter
            const int k0 = u0 / per, k1 = (u1 - 1) / per, s0 = 2 * k0 + (u0 == k0 * per ? 0 : 1);
            __syncthreads();
            if (tid == 0) {
                const unsigned seen = arrive_add(&a.arrive[s0]);
                is_last = seen == static_cast<unsigned>(k1 - k0);
                if (is_last) a.arrive[s0] = 0;
            }
            __syncthreads();
            if (is_last) {
                const long long step = static_cast<long long>(prow) * (D + 4);
                // Four dims of up to four rows per thread, two or four pieces at a time, all their loads in flight.
                constexpr int N = PIECES ? ROWS * D / 4 / (32 * NW) : 1, AT = N > 2 ? 2 : 4;
                const int row0 = tid / (D / 4), d = tid % (D / 4) * 4;
                float mx[N], lx[N];
                float4 y[N];
#pragma unroll
                for (int v = 0; v < N; ++v) mx[v] = -INFINITY, lx[v] = 0.0f, y[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                for (int k = k0; k <= k1; k += AT) {
                    float2 ml[AT][N];
                    float4 yk[AT][N];
#pragma unroll
                    for (int u = 0; u < AT; ++u) {
                        const int kk = min(k + u, k1);
                        const float *q = a.part + (kk == k0 ? s0 : 2 * kk) * step;
#pragma unroll
                        for (int v = 0; v < N; ++v) {
                            const int row = min(row0 + v * (128 * NW / D), rows - 1);
                            ml[u][v] = __ldcg(reinterpret_cast<const float2 *>(q + prow * D + 2 * row));
                            yk[u][v] = __ldcg(reinterpret_cast<const float4 *>(q + row * D + d));
                            if (k + u > k1) ml[u][v].x = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < AT; ++u)
#pragma unroll
                        for (int v = 0; v < N; ++v) {
                            const float mn = fmaxf(mx[v], ml[u][v].x);
                            if (mn == -INFINITY) continue;
                            const float f = ex2(mx[v] - mn), fk = ex2(ml[u][v].x - mn);
                            lx[v] = fmaf(lx[v], f, ml[u][v].y * fk);
                            y[v].x = fmaf(y[v].x, f, yk[u][v].x * fk);
                            y[v].y = fmaf(y[v].y, f, yk[u][v].y * fk);
                            y[v].z = fmaf(y[v].z, f, yk[u][v].z * fk);
                            y[v].w = fmaf(y[v].w, f, yk[u][v].w * fk);
                            mx[v] = mn;
                        }
                }
#pragma unroll
                for (int v = 0; v < N; ++v) {
                    const float inv = lx[v] != 0.0f ? 1.0f / lx[v] : 0.0f;
                    const int row = row0 + v * (128 * NW / D);
                    if (row < rows) put(h, row, d, make_float4(y[v].x * inv, y[v].y * inv, y[v].z * inv, y[v].w * inv));
                }
            }
        }
        x0 = x1;
    }
    if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(c.status, ST_KV8_BAD_PAGE);
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
    a.page_runs = static_cast<unsigned>(kv->nLayer * 2 * kv->nHead);
    a.k_run = static_cast<unsigned>(L * 2 * kv->nHead);
    a.part = w.part;
    a.arrive = w.arrive;
    const long long R = static_cast<long long>(a.G) * Tq;
    const int rows = R <= 8 ? 8 : 16, ck = kv8::HALF / kv->headDim;
    a.qtiles = static_cast<int>((R + rows - 1) / rows);
    const long long entries = static_cast<long long>(kv->nRow) * a.qtiles;
    const long long chunks = entries * kv->nHead * (a.max_len / ck + 2);  // at most
    if (entries > 0x7FFFFFFFll || R > 0x7FFFFFFFll - rows) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    // Plan. Units that fill the GPU have a CTA each: no prefix sum, no shared units. Groups of two rows (64 sequences x 12 heads
    // of 512 to 1023 keys: 23.3 us; four rows 30.3, two warps per row 24.2, equal pieces 30.9) as long as groups of four would
    // leave a third of the SMs' 12 warps empty, then of four (128 x 12 units of 640 to 700 keys: 14.4 us, of two 21.4; 256 x 12
    // of 150 to 300: 31.4 against 35.1). Windows, whose rows need not start together, and more query rows: one or two
    // warps per row by the same rule (128 x 12 units of 640 to 700 keys: 28.8 us with one, 33.5 with two). Fewer units: equal
    // pieces, four warps per CTA, which merge their rows before a piece's partials go through the work area.
    const long long units = entries * kv->nHead;
    const bool pieces = units < 3ll * ctx->num_sms && entries <= kv8::MAX_ENTRIES && chunks <= 0x3FFFFFFFll;
    const int warps = pieces ? kv8::NW_PIECES : units < 8ll * ctx->num_sms ? 2 : 1;
    a.entries = pieces ? static_cast<int>(entries) : 0;
    const int group = pieces || R > 4 || d_first ? 0 : warps == 1 && R <= 2 ? 4 : 2;
    const kv8::View c = kv8::view(kv, ctx->status);
    auto go = [&](auto kern, auto shape, int variant) {
        using SH = decltype(shape);
        bool *attr_done = &ctx->kv8_attr_done[variant];
        if (!*attr_done) {
            RelaxedCapture relaxed;
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SH::BYTES + (kv8::MAX_ENTRIES + 1) * 4) != cudaSuccess)
                return GPT2_B200_ECUDA;
            *attr_done = true;
        }
        const int smem = SH::BYTES + (a.entries + 1) * 4;
        // CTAs that are resident together: registers (the kernel's launch bounds) and 228 KB of shared memory, 1 KB of it per CTA.
        const int resident = std::min(SH::RESIDENT, 228 * 1024 / (smem + 1024 + 512));
        const int threads = 32 * (group ? kv8::NW_PIECES : warps);
        const dim3 grid =
            group    ? dim3((kv->nRow + group - 1) / group, kv->nHead)
            : pieces ? dim3(static_cast<unsigned>(std::min<long long>({static_cast<long long>(ctx->num_sms) * resident, kv8::MAX_PIECES,
                                                                        (chunks + warps - 1) / warps})))
                     : dim3(static_cast<unsigned>(entries), kv->nHead);
        kern<<<grid, threads, smem, stream>>>(c, a);
        return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
    };
    auto by_rows = [&](auto kind, auto dim) {
        constexpr int KIND = decltype(kind)::value, D = decltype(dim)::value;
        constexpr int base = (KIND == GPT2_KV8_INT8 ? 0 : 16) + (D == 64 ? 0 : 8);
        if (rows == 8) {
            if (group == 4) return go(kv8::k_kv8_attend<KIND, D, 8, 4, 4>, kv8::Shape<D, 8, 4>(), base);
            if (group == 2) return go(kv8::k_kv8_attend<KIND, D, 8, 4, 2>, kv8::Shape<D, 8, 4>(), base + 1);
            if (warps == 4) return go(kv8::k_kv8_attend<KIND, D, 8, 4, 0>, kv8::Shape<D, 8, 4>(), base + 2);
            if (warps == 2) return go(kv8::k_kv8_attend<KIND, D, 8, 2, 0>, kv8::Shape<D, 8, 2>(), base + 3);
            return go(kv8::k_kv8_attend<KIND, D, 8, 1, 0>, kv8::Shape<D, 8, 1>(), base + 4);
        }
        if (warps == 4) return go(kv8::k_kv8_attend<KIND, D, 16, 4, 0>, kv8::Shape<D, 16, 4>(), base + 5);
        if (warps == 2) return go(kv8::k_kv8_attend<KIND, D, 16, 2, 0>, kv8::Shape<D, 16, 2>(), base + 6);
        return go(kv8::k_kv8_attend<KIND, D, 16, 1, 0>, kv8::Shape<D, 16, 1>(), base + 7);
    };
    auto by_dim = [&](auto kind) {
        return kv->headDim == 64 ? by_rows(kind, std::integral_constant<int, 64>()) : by_rows(kind, std::integral_constant<int, 128>());
    };
    return kv->kind == GPT2_KV8_INT8 ? by_dim(std::integral_constant<int, GPT2_KV8_INT8>())
                                     : by_dim(std::integral_constant<int, GPT2_KV8_E4M3>());
}
