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

// Four pairs of whole numbers c (LEAST) or c - 8 out of a word, exact in fp16: a code under the exponent of 1024 is
// 1024 + c, or 1024 + 16 c from a nibble further up.
template <bool LEAST>
__device__ __forceinline__ void codes_of(uint32_t w, __half2 (&h)[4]) {
    constexpr uint32_t magic = 0x64006400u;
    const __half2 off = __float2half2_rn(LEAST ? -1024.0f : -1032.0f), off16 = __float2half2_rn(LEAST ? -64.0f : -72.0f);
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    uint32_t p[4];
    const uint32_t up = w >> 8;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(p[0]) : "r"(w), "r"(magic));
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(p[1]) : "r"(w), "r"(magic));
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(p[2]) : "r"(up), "r"(magic));
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(p[3]) : "r"(up), "r"(magic));
    h[0] = __hadd2(*reinterpret_cast<__half2 *>(&p[0]), off);
    h[1] = __hfma2(*reinterpret_cast<__half2 *>(&p[1]), sixteenth, off16);
    h[2] = __hadd2(*reinterpret_cast<__half2 *>(&p[2]), off);
    h[3] = __hfma2(*reinterpret_cast<__half2 *>(&p[3]), sixteenth, off16);
}

// The values of a word's 8 codes, one rounding each; s and l hold the scale and the least value twice.
template <bool LEAST>
__device__ __forceinline__ void values_of(uint32_t w, __half2 s, __half2 l, uint32_t (&v)[4]) {
    __half2 h[4];
    codes_of<LEAST>(w, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 y = LEAST ? __hfma2(h[i], s, l) : __hmul2(h[i], s);
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

struct Plan {
    GPT2W4 w;
    const __half *x;
    long long ldx;
    Dest d;
    bool pdl;
};

bool shape_ok(const GPT2W4 *w);    // sizes
bool weight_ok(const GPT2W4 *w);   // and pointers
int plan(Plan *pl, int epi, const GPT2W4 &w, const __half *x, long long ldx, int B, const __half *bias, __half *out, long long ldo);
int keys_of(const GPT2W4 &w, int B);  // argmax keys per row that a plan of EPI_HEAD writes
int prepare(const Plan &pl);          // kernel attributes, so that a capture finds them set
int launch(const Plan &pl, cudaStream_t stream);

}  // namespace w4
}  // namespace b200
