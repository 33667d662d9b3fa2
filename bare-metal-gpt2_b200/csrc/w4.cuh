// w4.cuh — 4-bit weights with group scales (internal): the format, its conversion in registers, and the product's
// interface to the decode step.
//
// A weight W[N][K] is held as codes 0..15, 8 to a 32-bit word, row after row; every `group` (32, 64 or 128)
// neighbouring k of a row have one fp16 scale s and, in the form with `least`, one fp16 smallest value l. A code c
// stands for the fp16 nearest to c * s + l, or (c - 8) * s: the same rounding as an fp16 checkpoint of these values
// has, 2^-12 of a weight against a code's step of 2^-4, and what lets the tensor cores take the weights as they are
// (scaling partial sums in fp32 instead would need the sums of every group apart).
//   - Element 2 i of a word lies in bits 4 i .. 4 i + 3, element 2 i + 1 in bits 16 + 4 i ..: a mask and an or give two
//     neighbouring elements as the halves of a register, in the order that the matrix instructions take them.
//   - scale and least are [K / group][N]: the rows of a tile are neighbours.
#pragma once
#include "common.cuh"
#include "linear.cuh"
#include "ptx.cuh"

namespace b200 {
namespace w4 {

// The values of a word's codes, one rounding each. A code masked out at bits 6..9 of a half is the subnormal c * 2^-18, exact, so
// rn(c * s + l) is one fused multiply-add with s * 2^18, and rn((c - 8) * s) is one with -8 s: 8 shifts and masks and 4 fused
// operations for 8 codes. s * 2^18 is a number for s < 0.25, which weights of models keep by far; where some scale of the
// warp is larger (or negative, or not finite: `big`) the codes are made whole numbers first. The same bits either way. Putting a code under the
// exponent of 1024 instead needs the second operation always: 47 cycles per 2048 codes on an SM against 38, where reading them from HBM
// takes 47.
__device__ __forceinline__ bool big_scale(uint32_t bits) { return bits >= 0x3400u; }  // fp16 bits: 0.25 and above, negative, NaN

struct Scale {
    __half2 s, l;
};
template <bool LEAST, bool BIG>
__device__ __forceinline__ Scale scale_of(uint32_t s_bits, uint32_t l_bits) {
    const __half s = __ushort_as_half(static_cast<unsigned short>(s_bits));
    const __half2 s2 = __half2half2(s), up = __float2half2_rn(512.0f);
    const __half2 l2 = LEAST ? __half2half2(__ushort_as_half(static_cast<unsigned short>(l_bits))) : __hmul2(s2, __float2half2_rn(-8.0f));
    if (!BIG) return {__hmul2(__hmul2(s2, up), up), l2};
    return {s2, LEAST ? l2 : __float2half2_rn(0.0f)};
}

template <bool LEAST, bool BIG>
__device__ __forceinline__ void values_of(uint32_t w, const Scale &sc, uint32_t (&v)[4]) {
    constexpr uint32_t mask = 0x03C003C0u;
    const uint32_t p[4] = {(w << 6) & mask, (w << 2) & mask, (w >> 2) & mask, (w >> 6) & mask};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 h = *reinterpret_cast<const __half2 *>(&p[i]);
        if (BIG) h = __hfma2(__hmul2(h, __float2half2_rn(32768.0f)), __float2half2_rn(8.0f), __float2half2_rn(LEAST ? 0.0f : -8.0f));
        const __half2 y = __hfma2(h, sc.s, sc.l);
        v[i] = *reinterpret_cast<const uint32_t *>(&y);
    }
}

// What happens to acc = sum + bias of feature n and row b. One rounding to fp16 at the end of each.
struct Dest {
    int epi;             // lin::Epi
    int B, N;
    const __half *bias;  // [N] or null
    __half *out;         // [B][ldo]; EPI_HEAD: logits, may be null
    long long ldo;
    const __half *resid;  // EPI_RESID: [B][ldr], may be out
    long long ldr;
    // EPI_QKV: K and V columns also go to sequence b's slabs [H][maxT][64] at d_pos[b]
    __half *const *k_dst;
    __half *const *v_dst;
    const int *d_pos;
    int maxT, E;
    // EPI_HEAD: argmax keys [B][keys]
    unsigned long long *amax;
    int keys;
    unsigned *status;
};

struct RowParams {
    const uint8_t *codes;
    const __half *scale, *least;
    int K, shift;  // log2 of the group
    const __half *x;
    long long ldx;
    int tiles, steps;  // tiles; steps of a warp per tile
    int ahead;                // codes are fetched before x
    Dest d;
};

struct TcParams {
    const __half *scale, *least;
    int K, shift;            // shift: log2 of the group
    int stages, cs, tiles;   // per tile; CTAs that share a tile's k; tiles
    int x_ring, bpad, nacc;  // stages of x in flight; columns; accumulators
    int push, share;         // split k: sums are pushed to the CTA that adds them (else pulled); columns that each adds
    Dest d;
    unsigned long long timeout_ns;
};

// A launch that was thought out: which kernel, how it is split, its tensor maps.
struct Plan {
    CUtensorMap tm_w, tm_x;
    RowParams rows;  // few
    TcParams tc;     // else
    Dest d;
    bool few, pdl;  // pdl: a programmatic dependent of the kernel before it
    const void *kernel;
    dim3 grid;
    int threads, cluster;
    size_t smem;
};

bool weight_ok(const GPT2W4 *w);  // sizes and pointers
// resid and ldr: EPI_RESID's. Returns a GPT2_B200_* code; d's fields of EPI_QKV and EPI_HEAD are the caller's to fill in.
int plan(Plan *pl, int epi, const GPT2W4 &w, const __half *x, long long ldx, int B, const __half *bias, __half *out, long long ldo, const __half *resid, long long ldr);
// d: the plan's own, or it with other pointers. The plan stays as it is.
int launch(const Plan &pl, const Dest &d, cudaStream_t stream);
inline int launch(const Plan &pl, cudaStream_t stream) { return launch(pl, pl.d, stream); }

}  // namespace w4
}  // namespace b200
