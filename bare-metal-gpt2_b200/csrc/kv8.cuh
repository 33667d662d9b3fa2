// kv8.cuh — the paged 8-bit KV cache (internal): checks, addresses, code conversions, work area.
//
// One page holds `page` positions of every layer and head, so that sharing, copying and moving a page
// is one table entry and one contiguous run of bytes. A (page, layer, K|V, head) run of page * headDim
// code bytes is what the attention streams; its page / block scales lie apart in `scale`.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {
namespace kv8 {

constexpr int MAX_ROWS = 1024;  // one thread per row in the page planner

// What the kernels get of a cache.
struct View {
    uint8_t *data;
    float *scale;
    int *ref, *table, *len;
    int nPages, nRow, maxPages, nLayer, nHead, D, page, block, page_shift, block_shift;
    unsigned *status;

};

// Work area: counters (zero between calls), then the planner's lists, then the attention's partials.
struct Work {
    unsigned *misc;      // [64] planner counters
    unsigned *arrive;    // [attend_max_ctas()] split-merge arrivals, one per tile of query rows
    int4 *copies;        // [nRow] (source, destination, positions, unused)
    int *list;           // [nPages] free pages found / new id of a moved page
    int2 *moves;         // [nPages / 2] (source, destination) of a compaction
    float *part;         // split partials
    size_t bytes;
};

inline int shift_of(int v) { return v == 16 ? 4 : v == 32 ? 5 : v == 64 ? 6 : v == 128 ? 7 : -1; }

// CTAs up to which an attention launch splits keys (see the plan in kv8_attend.cu).
int attend_max_ctas();
constexpr int ATT_TILE = 16;  // query rows (tokens x heads of a group) per CTA

inline bool shape_ok(const GPT2KV8Cache *kv) {
    return kv && kv->nPages >= 1 && kv->nRow >= 1 && kv->nRow <= MAX_ROWS && kv->maxPages >= 1 &&
           kv->nLayer >= 1 && kv->nHead >= 1 && (kv->headDim == 64 || kv->headDim == 128) &&
           shift_of(kv->page) > 0 && shift_of(kv->block) > 0 && kv->block <= kv->page &&
           static_cast<long long>(kv->maxPages) * kv->page <= 0x3FFFFFFFll && kv->nHead <= 65535 &&
           static_cast<long long>(kv->nRow) * kv->maxPages <= 0x7FFFFFFFll &&
           // rows of codes (a position of one page, layer, K|V and head) are counted in 32 bits: 256 GB of them and more
           static_cast<double>(kv->nPages) * kv->nLayer * 2.0 * kv->nHead * kv->page < 4294967296.0 &&
           (kv->kind == GPT2_KV8_INT8 || kv->kind == GPT2_KV8_E4M3);
}

// The arrival counters have the same place and size for every call on a cache (they are zero between
// calls): only launches of at most attend_max_ctas() CTAs split their keys, so as many tiles at most merge.
inline Work work_layout(const GPT2KV8Cache *kv, int Hq, int Tq) {
    Work w;
    auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    const size_t group_rows = static_cast<size_t>(Tq) * (Hq / kv->nHead);
    const size_t rows = group_rows < ATT_TILE ? group_rows : ATT_TILE;
    const size_t o_arr = 256, o_cop = o_arr + up(attend_max_ctas() * 4ull), o_list = o_cop + up(kv->nRow * sizeof(int4));
    const size_t o_mov = o_list + up(static_cast<size_t>(kv->nPages) * 4);
    const size_t o_part = o_mov + up(static_cast<size_t>(kv->nPages / 2 + 1) * sizeof(int2));
    char *b = static_cast<char *>(kv->work);
    w.misc = reinterpret_cast<unsigned *>(b);
    w.arrive = reinterpret_cast<unsigned *>(b + o_arr);
    w.copies = reinterpret_cast<int4 *>(b + o_cop);
    w.list = reinterpret_cast<int *>(b + o_list);
    w.moves = reinterpret_cast<int2 *>(b + o_mov);
    w.part = reinterpret_cast<float *>(b + o_part);
    w.bytes = o_part + up(attend_max_ctas() * rows * (kv->headDim + 4) * sizeof(float));
    return w;
}

inline bool aligned(const void *p, uintptr_t n = 16) { return p && (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Full check of a descriptor; GPT2_B200_OK or _EINVAL, before any CUDA call.
inline int check(const GPT2KV8Cache *kv) {
    if (!shape_ok(kv) || !aligned(kv->data) || !aligned(kv->scale) || !aligned(kv->ref) ||
        !aligned(kv->table) || !aligned(kv->len) || !aligned(kv->work))
        return GPT2_B200_EINVAL;
    return GPT2_B200_OK;
}

inline View view(const GPT2KV8Cache *kv, unsigned *status) {
    View v;
    v.data = static_cast<uint8_t *>(kv->data);
    v.scale = kv->scale;
    v.ref = kv->ref;
    v.table = kv->table;
    v.len = kv->len;
    v.nPages = kv->nPages;
    v.nRow = kv->nRow;
    v.maxPages = kv->maxPages;
    v.nLayer = kv->nLayer;
    v.nHead = kv->nHead;
    v.D = kv->headDim;
    v.page = kv->page;
    v.block = kv->block;
    v.page_shift = shift_of(kv->page);
    v.block_shift = shift_of(kv->block);
    v.status = status;
    return v;
}

// Counts this CTA in at a counter in global memory. Called by one thread behind a CTA barrier and before another: what the
// CTA wrote before is visible to the CTA that counts last, and what the others wrote is visible to this one (release and
// acquire at GPU scope; the two barriers carry both to the CTA's other threads).
__device__ __forceinline__ unsigned arrive_add(unsigned *p) {
    unsigned v;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// ---------------------------------------------------------------- codes
template <int KIND>
__device__ __forceinline__ float qmax() {
    return KIND == GPT2_KV8_INT8 ? 127.0f : 448.0f;
}
template <int KIND>
__device__ __forceinline__ float decode(unsigned c) {
    if (KIND == GPT2_KV8_INT8) return static_cast<float>(static_cast<signed char>(c));
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3)));
}
// The nearest code of x (ties to even), clamped to the type's range.
template <int KIND>
__device__ __forceinline__ unsigned encode(float x) {
    if (KIND == GPT2_KV8_INT8)
        return static_cast<unsigned>(__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f))) & 0xFFu;
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace kv8
}  // namespace b200
