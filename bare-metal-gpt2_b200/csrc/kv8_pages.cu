// kv8_pages.cu — the pages of the 8-bit cache: allocation, reset, reorder (fork, free, copy on write,
// reserve) and compaction.
//
// A reorder is planned by one CTA (counts, ranks and the scan for free pages are sequential in row
// order by definition, so the page ids do not depend on timing) and its page copies run on the
// whole GPU. Compaction is a scan of the reference counts, then copies between disjoint pages.
#include <cstdio>

#include "kv8.cuh"

namespace b200 {
namespace kv8 {

constexpr int PLAN_NT = 1024;
enum Misc { M_COPIES = 0, M_LIVE = 1 };

// Exclusive prefix sum of v over the CTA's PLAN_NT threads; *total receives the sum.
__device__ int block_scan(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();  // warp_sums may still be read from a previous call
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, w, o);
            if (lane >= o) w += u;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *total = warp_sums[31];
    return s - v + (warp ? warp_sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(PLAN_NT) k_kv8_plan(const View c, const Work w, const int *parent, int advance,
                                                      int reserve) {
    __shared__ int sums[32];
    __shared__ int tail_page[MAX_ROWS];
    const int tid = threadIdx.x, M = c.maxPages, cap = M << c.page_shift;
    // the state before: table0 (copied by the caller), len0 = len + advance
    if (tid < c.nRow) {
        long long n = static_cast<long long>(c.len[tid]) + advance;
        if (n < 0 || n > cap) {
            atomicOr(c.status, ST_KV8_BAD_LEN);
            n = n < 0 ? 0 : cap;
        }
        w.len0[tid] = static_cast<int>(n);
    }
    __syncthreads();
    // drop every old hold, take every new one
    for (long long e = tid; e < static_cast<long long>(c.nRow) * M; e += PLAN_NT) {
        const int old = w.table0[e];
        if (old >= 0 && old < c.nPages) atomicSub(&c.ref[old], 1);
    }
    for (long long e = tid; e < static_cast<long long>(c.nRow) * M; e += PLAN_NT) {
        const int r = static_cast<int>(e / M), i = static_cast<int>(e - static_cast<long long>(r) * M);
        int from = parent ? parent[r] : r;
        if (from < -1 || from >= c.nRow) {
            if (i == 0) atomicOr(c.status, ST_KV8_BAD_PARENT);
            from = -1;
        }
        int p = -1;
        if (from >= 0 && i < (w.len0[from] + c.page - 1) >> c.page_shift) {
            p = w.table0[static_cast<long long>(from) * M + i];
            if (p < 0 || p >= c.nPages) {
                atomicOr(c.status, ST_KV8_BAD_PAGE);
                p = -1;
            } else {
                atomicAdd(&c.ref[p], 1);
            }
        }
        c.table[e] = p;
    }
    __syncthreads();
    // what each row needs
    int n = 0, held = 0, last = -1, copy = 0, grow = 0;
    if (tid < c.nRow) {
        const int from = parent ? parent[tid] : tid;
        n = from >= 0 && from < c.nRow ? w.len0[from] : 0;
        c.len[tid] = n;
        held = (n + c.page - 1) >> c.page_shift;
        if (reserve > 0 && (n & (c.page - 1))) last = c.table[static_cast<long long>(tid) * M + held - 1];
        tail_page[tid] = last;
        const long long want = (static_cast<long long>(n) + reserve + c.page - 1) >> c.page_shift;
        if (want > M) atomicOr(c.status, ST_KV8_NO_PAGE);
        grow = static_cast<int>(want > M ? M : want) - held;
    }
    __syncthreads();
    if (last >= 0) {
        int before = 0;  // earlier rows that continue in the same page
        for (int q = 0; q < tid; ++q) before += tail_page[q] == last;
        copy = before < __ldcg(&c.ref[last]) - 1;
    }
    int total;
    const int off = block_scan(copy + grow, sums, &total);
    // the lowest-numbered free pages
    int found = 0;
    for (int base = 0; base < c.nPages && found < total; base += PLAN_NT) {
        const int p = base + tid;
        const int free_page = p < c.nPages && __ldcg(&c.ref[p]) == 0;
        int some;
        const int at = found + block_scan(free_page, sums, &some);
        if (free_page && at < total) w.list[at] = p;
        found += some;
    }
    __syncthreads();
    int copies;
    const int cat = block_scan(copy, sums, &copies);
    if (tid < c.nRow) {
        int *row = c.table + static_cast<long long>(tid) * M;
        if (copy) {
            int p = -1;
            if (off < found) {
                p = w.list[off];
                c.ref[p] = 1;
            } else {
                atomicOr(c.status, ST_KV8_NO_PAGE);
            }
            row[held - 1] = p;
            atomicSub(&c.ref[last], 1);
            w.copies[cat] = make_int4(last, p, n & (c.page - 1), 0);
        }
        for (int i = 0; i < grow; ++i) {
            if (off + copy + i >= found) {
                atomicOr(c.status, ST_KV8_NO_PAGE);
                break;
            }
            const int p = w.list[off + copy + i];
            c.ref[p] = 1;
            row[held + i] = p;
        }
    }
    if (tid == 0) w.misc[M_COPIES] = copies;
}

// The filled part of each copied page: every layer, K|V and head, and the scales of its blocks.
__global__ void __launch_bounds__(256) k_kv8_copy(const View c, const Work w) {
    const int copies = static_cast<int>(w.misc[M_COPIES]);
    const int runs = c.nLayer * 2 * c.nHead, nb = c.page >> c.block_shift;
    for (long long u = blockIdx.x; u < static_cast<long long>(copies) * runs; u += gridDim.x) {
        const int4 cp = w.copies[u / runs];
        if (cp.y < 0) continue;
        const long long i = u % runs, src = static_cast<long long>(cp.x) * runs + i, dst = static_cast<long long>(cp.y) * runs + i;
        const uint4 *s = reinterpret_cast<const uint4 *>(c.data + (src << c.page_shift) * c.D);
        uint4 *d = reinterpret_cast<uint4 *>(c.data + (dst << c.page_shift) * c.D);
        for (int x = threadIdx.x; x < cp.z * c.D / 16; x += 256) d[x] = s[x];
        if (static_cast<int>(threadIdx.x) < (cp.z + c.block - 1) >> c.block_shift)
            c.scale[dst * nb + threadIdx.x] = c.scale[src * nb + threadIdx.x];
    }
}

// Compaction: list[p] = new id of page p (itself below live); copies between disjoint pages.
__global__ void __launch_bounds__(PLAN_NT) k_kv8_compact_plan(const View c, const Work w, int *d_live) {
    __shared__ int sums[32];
    const int tid = threadIdx.x;
    int mine = 0, live;
    for (int p = tid; p < c.nPages; p += PLAN_NT) mine += c.ref[p] > 0;
    block_scan(mine, sums, &live);
    // list[0..]: the holes below live in ascending order
    int holes = 0;
    for (int base = 0; base < live; base += PLAN_NT) {
        const int p = base + tid;
        const int hole = p < live && c.ref[p] <= 0;
        int some;
        const int at = holes + block_scan(hole, sums, &some);
        if (hole) w.list[at] = p;
        holes += some;
        __syncthreads();
    }
    int seen = 0;
    for (int base = live & ~(PLAN_NT - 1); base < c.nPages; base += PLAN_NT) {
        const int p = base + tid;
        const int move = p >= live && p < c.nPages && c.ref[p] > 0;
        int some;
        const int at = seen + block_scan(move, sums, &some);
        // list[p], p >= live: the new id. Fewer than live holes, so the map does not overlap their list.
        if (p >= live && p < c.nPages) {
            const int to = move ? w.list[at] : -1;
            if (move) {
                c.ref[to] = c.ref[p];
                c.ref[p] = 0;
            }
            w.list[p] = to;
        }
        seen += some;
    }
    if (tid == 0) {
        w.misc[M_LIVE] = live;
        if (d_live) *d_live = live;
    }
}

__global__ void __launch_bounds__(256) k_kv8_compact_move(const View c, const Work w) {
    const int live = static_cast<int>(w.misc[M_LIVE]);
    const long long entries = static_cast<long long>(c.nRow) * c.maxPages;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < entries; e += gridDim.x * 256ll) {
        const int p = c.table[e];
        if (p >= live && p < c.nPages) c.table[e] = w.list[p];
    }
    const int runs = c.nLayer * 2 * c.nHead, nb = c.page >> c.block_shift;
    const long long bytes = static_cast<long long>(runs) * c.page * c.D, scales = static_cast<long long>(runs) * nb;
    for (int p = live + blockIdx.x; p < c.nPages; p += gridDim.x) {
        const int to = w.list[p];
        if (to < 0) continue;
        const uint4 *s = reinterpret_cast<const uint4 *>(c.data + p * bytes);
        uint4 *d = reinterpret_cast<uint4 *>(c.data + to * bytes);
        for (long long x = threadIdx.x; x < bytes / 16; x += 256) d[x] = s[x];
        for (long long x = threadIdx.x; x < scales; x += 256) c.scale[to * scales + x] = c.scale[p * scales + x];
    }
}

__global__ void k_kv8_reset(const View c) {
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i < c.nPages) c.ref[i] = 0;
    if (i < c.nRow) c.len[i] = 0;
    if (i < static_cast<long long>(c.nRow) * c.maxPages) c.table[i] = -1;
}

static size_t up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

}  // namespace kv8
}  // namespace b200

using namespace b200;

extern "C" {

size_t gpt2_kv8_work_bytes_b200(const GPT2KV8Cache *kv, int Hq, int Tq) {
    if (!kv8::shape_ok(kv) || Hq < 1 || Hq % kv->nHead || Tq < 1) return 0;
    return kv8::work_layout(kv, Hq, Tq).bytes;
}

int gpt2_kv8_reset_b200(const GPT2KV8Cache *kv, cudaStream_t stream) {
    if (kv8::check(kv) != GPT2_B200_OK) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    const long long n = std::max<long long>(kv->nPages, static_cast<long long>(kv->nRow) * std::max(kv->maxPages, 1));
    kv8::k_kv8_reset<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(kv8::view(kv, ctx->status));
    if (cudaGetLastError() != cudaSuccess || cudaMemsetAsync(kv->work, 0, kv->work_bytes, stream) != cudaSuccess)
        return GPT2_B200_ECUDA;
    return GPT2_B200_OK;
}

int gpt2_kv8_alloc_b200(GPT2KV8Cache *kv, int Hq, int Tq) {
    if (!kv) return 1;
    kv->data = kv->work = nullptr;
    kv->scale = nullptr;
    kv->ref = kv->table = kv->len = nullptr;
    kv->work_bytes = gpt2_kv8_work_bytes_b200(kv, Hq, Tq);
    if (!kv->work_bytes) return 1;
    const size_t runs = static_cast<size_t>(kv->nPages) * kv->nLayer * 2 * kv->nHead;
    const size_t data = kv8::up(runs * kv->page * kv->headDim), scale = kv8::up(runs * (kv->page / kv->block) * 4);
    const size_t ref = kv8::up(static_cast<size_t>(kv->nPages) * 4), len = kv8::up(static_cast<size_t>(kv->nRow) * 4);
    const size_t table = kv8::up(static_cast<size_t>(kv->nRow) * kv->maxPages * 4);
    const size_t total = data + scale + ref + len + table + kv8::up(kv->work_bytes);
    size_t free_b = 0, total_b = 0;
    if (cudaMemGetInfo(&free_b, &total_b) != cudaSuccess) return 1;
    const size_t headroom = static_cast<size_t>(64) << 20;  // the fp16 arena's refusal rule
    if (total + headroom > free_b) {
        fprintf(stderr,
                "[gpt2_b200] 8-bit KV cache of %zu bytes not allocated: %zu bytes free on the device, and %zu must stay "
                "free after it\n",
                total, free_b, headroom);
        return 1;
    }
    char *p = nullptr;
    if (cudaMalloc(&p, total) != cudaSuccess) return 1;
    kv->data = p;
    kv->scale = reinterpret_cast<float *>(p + data);
    kv->ref = reinterpret_cast<int *>(p + data + scale);
    kv->len = reinterpret_cast<int *>(p + data + scale + ref);
    kv->table = reinterpret_cast<int *>(p + data + scale + ref + len);
    kv->work = p + data + scale + ref + len + table;
    if (gpt2_kv8_reset_b200(kv, 0) != GPT2_B200_OK || cudaStreamSynchronize(0) != cudaSuccess) {
        gpt2_kv8_free_b200(kv);
        return 1;
    }
    return 0;
}

void gpt2_kv8_free_b200(GPT2KV8Cache *kv) {
    if (kv && kv->data) {
        cudaFree(kv->data);  // one allocation holds all six arrays
        kv->data = kv->work = nullptr;
        kv->scale = nullptr;
        kv->ref = kv->table = kv->len = nullptr;
    }
}

int gpt2_kv8_reorder_b200(const GPT2KV8Cache *kv, const int *parent, int advance, int reserve, cudaStream_t stream) {
    if (kv8::check(kv) != GPT2_B200_OK || advance < 0 || reserve < 0 || kv->work_bytes < kv8::work_layout(kv, kv->nHead, 1).bytes)
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    const kv8::Work w = kv8::work_layout(kv, kv->nHead, 1);
    const kv8::View c = kv8::view(kv, ctx->status);
    if (cudaMemcpyAsync(w.table0, kv->table, static_cast<size_t>(kv->nRow) * kv->maxPages * 4, cudaMemcpyDeviceToDevice, stream) !=
        cudaSuccess)
        return GPT2_B200_ECUDA;
    kv8::k_kv8_plan<<<1, kv8::PLAN_NT, 0, stream>>>(c, w, parent, advance, reserve);
    kv8::k_kv8_copy<<<ctx->num_sms * 8, 256, 0, stream>>>(c, w);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

int gpt2_kv8_compact_b200(const GPT2KV8Cache *kv, int *d_live, cudaStream_t stream) {
    if (kv8::check(kv) != GPT2_B200_OK || kv->work_bytes < kv8::work_layout(kv, kv->nHead, 1).bytes) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    const kv8::Work w = kv8::work_layout(kv, kv->nHead, 1);
    const kv8::View c = kv8::view(kv, ctx->status);
    kv8::k_kv8_compact_plan<<<1, kv8::PLAN_NT, 0, stream>>>(c, w, d_live);
    kv8::k_kv8_compact_move<<<ctx->num_sms * 8, 256, 0, stream>>>(c, w);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // extern "C"
