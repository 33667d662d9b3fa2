// kv8_pages.cu — the pages of the 8-bit cache: allocation, reset, reorder (fork, free, copy on write,
// reserve) and compaction.
//
// Measured: 128 rows of 63 pages, 64 copies of half-filled 295 KB pages: 15.6 us, latency-bound (the plan's scans depend
// on each other, the copies on the plan); compaction that moves 300 such pages: 31.5 us, 25.8 of it at HBM's rate.
//
// A reorder is planned by one CTA (counts, ranks and the scan for free pages are sequential in row
// order by definition, so the page ids do not depend on timing) and its page copies run on the
// whole GPU. Compaction is a scan of the reference counts, then copies between disjoint pages.
#include <algorithm>
#include <cstdio>

#include "kv8.cuh"
#include "ptx.cuh"

namespace b200 {
namespace kv8 {

constexpr int PLAN_NT = 1024;
constexpr int ENTRIES = 8;  // table entries per thread and batch
enum Misc { M_COPIES = 0, M_LIVE = 1, M_MOVES = 2 };

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
    __shared__ int len0[MAX_ROWS], from0[MAX_ROWS];
    __shared__ __align__(16) int tail_page[MAX_ROWS];
    grid_launch_dependents();  // the copies' CTAs wait for this one's end
    const int tid = threadIdx.x, M = c.maxPages, cap = M << c.page_shift;
    if (tid < c.nRow) {
        long long n = static_cast<long long>(c.len[tid]) + advance;
        if (n < 0 || n > cap) {
            atomicOr(c.status, ST_KV8_BAD_LEN);
            n = n < 0 ? 0 : cap;
        }
        int from = parent ? parent[tid] : tid;
        if (from < -1 || from >= c.nRow) {
            atomicOr(c.status, ST_KV8_BAD_PARENT);
            from = -1;
        }
        len0[tid] = static_cast<int>(n);
        from0[tid] = from;
    }
    __syncthreads();
    // Every entry's old and new page. A row's new entry comes from another row's old one in the same column, so a batch of
    // whole columns is read before any of it is written. Beams share most pages with their parent: where old and
    // new are the same page nothing is done.
    const int cols = max(1, min(M, PLAN_NT * ENTRIES / c.nRow));
    for (int c0 = 0; c0 < M; c0 += cols) {
        const int width = min(cols, M - c0), total = width * c.nRow;
        int old_page[ENTRIES], new_page[ENTRIES], at[ENTRIES];
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j) {
            const int e = tid + j * PLAN_NT;
            at[j] = -1;
            if (e < total) {
                const int r = e / width, i = c0 + e - r * width, from = from0[r];
                at[j] = r * M + i;
                old_page[j] = c.table[at[j]];
                new_page[j] = -1;
                if (from >= 0 && i < (len0[from] + c.page - 1) >> c.page_shift) {
                    new_page[j] = c.table[from * M + i];
                    if (new_page[j] < 0 || new_page[j] >= c.nPages) {
                        atomicOr(c.status, ST_KV8_BAD_PAGE);
                        new_page[j] = -1;
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ENTRIES; ++j)
            if (at[j] >= 0 && old_page[j] != new_page[j]) {
                if (old_page[j] >= 0 && old_page[j] < c.nPages) atomicSub(&c.ref[old_page[j]], 1);
                if (new_page[j] >= 0) atomicAdd(&c.ref[new_page[j]], 1);
                c.table[at[j]] = new_page[j];
            }
        __syncthreads();
    }
    // what each row needs
    int n = 0, held = 0, last = -1, copy = 0, grow = 0;
    if (tid < c.nRow) {
        n = from0[tid] >= 0 ? len0[from0[tid]] : 0;
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
        const int holds = __ldcg(&c.ref[last]);
        if (holds > 1) {
            int before = 0;  // earlier rows that continue in the same page
            const int4 *t4 = reinterpret_cast<const int4 *>(tail_page);
            for (int q = 0; q < tid >> 2; ++q) {
                const int4 z = t4[q];
                before += (z.x == last) + (z.y == last) + (z.z == last) + (z.w == last);
            }
            for (int q = tid & ~3; q < tid; ++q) before += tail_page[q] == last;
            copy = before < holds - 1;
        }
    }
    int total;
    const int off = block_scan(copy + grow, sums, &total);
    // the lowest-numbered free pages, four per thread and step
    int found = 0;
    for (int base = 0; base < c.nPages && found < total; base += 4 * PLAN_NT) {
        const int p0 = base + 4 * tid;
        int is_free[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            is_free[i] = p0 + i < c.nPages && __ldcg(&c.ref[p0 + i]) == 0;
            mine += is_free[i];
        }
        int some;
        int at = found + block_scan(mine, sums, &some);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (is_free[i]) {
                if (at < total) w.list[at] = p0 + i;
                ++at;
            }
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

// The filled part of each copied page: every layer, K|V and head, and the scales of its blocks. A warp per run.
__global__ void __launch_bounds__(256) k_kv8_copy(View c, Work w) {
    grid_dependency_wait();
    const int copies = static_cast<int>(__ldcg(&w.misc[M_COPIES]));
    const int runs = c.nLayer * 2 * c.nHead, sub = c.page_shift - c.block_shift, lane = threadIdx.x & 31;
    const long long items = static_cast<long long>(copies) * runs;
    for (long long u = blockIdx.x * 8 + (threadIdx.x >> 5); u < items; u += gridDim.x * 8) {
        const int which = static_cast<int>(u / runs), i = static_cast<int>(u - static_cast<long long>(which) * runs);
        const int4 cp = __ldcg(&w.copies[which]);
        if (cp.y < 0) continue;
        const unsigned src = static_cast<unsigned>(cp.x) * runs + i, dst = static_cast<unsigned>(cp.y) * runs + i;
        const uint4 *s = reinterpret_cast<const uint4 *>(c.data + (static_cast<size_t>(src) << c.page_shift) * c.D);
        uint4 *d = reinterpret_cast<uint4 *>(c.data + (static_cast<size_t>(dst) << c.page_shift) * c.D);
        const int n = cp.z * c.D / 16;
        for (int x = lane; x < n; x += 128) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x + 32 * j < n) v[j] = s[x + 32 * j];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (x + 32 * j < n) d[x + 32 * j] = v[j];
        }
        if (lane < (cp.z + c.block - 1) >> c.block_shift) c.scale[(dst << sub) + lane] = c.scale[(src << sub) + lane];
    }
}

// Compaction: list[p] = new id of page p (itself below live); copies between disjoint pages.
__global__ void __launch_bounds__(PLAN_NT) k_kv8_compact_plan(const View c, const Work w, int *d_live) {
    __shared__ int sums[32];
    grid_launch_dependents();
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
    for (int base = live; base < c.nPages; base += PLAN_NT) {
        const int p = base + tid;
        const int move = p < c.nPages && c.ref[p] > 0;
        int some;
        const int at = seen + block_scan(move, sums, &some);
        // list[p], p >= live: the new id. Fewer than live holes, so the map does not overlap their list.
        if (p < c.nPages) {
            const int to = move ? w.list[at] : -1;
            if (move) {
                c.ref[to] = c.ref[p];
                c.ref[p] = 0;
                w.moves[at] = make_int2(p, to);
            }
            w.list[p] = to;
        }
        seen += some;
    }
    if (tid == 0) {
        w.misc[M_LIVE] = live;
        w.misc[M_MOVES] = seen;
        if (d_live) *d_live = live;
    }
}

// The tables' new ids, then the moved pages' bytes, a CTA per SEGMENT of a page at a time.
constexpr int SEGMENT = 16384;
__global__ void __launch_bounds__(256) k_kv8_compact_move(View c, Work w) {
    grid_dependency_wait();
    const int live = static_cast<int>(__ldcg(&w.misc[M_LIVE])), moves = static_cast<int>(__ldcg(&w.misc[M_MOVES]));
    const long long entries = static_cast<long long>(c.nRow) * c.maxPages;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < entries; e += gridDim.x * 256ll) {
        const int p = c.table[e];
        if (p >= live && p < c.nPages) c.table[e] = __ldcg(&w.list[p]);
    }
    const int runs = c.nLayer * 2 * c.nHead;
    const long long bytes = static_cast<long long>(runs) * c.page * c.D, scales = static_cast<long long>(runs) << (c.page_shift - c.block_shift);
    const long long segs = (bytes + SEGMENT - 1) / SEGMENT;
    for (long long u = blockIdx.x; u < moves * segs; u += gridDim.x) {
        const int m = static_cast<int>(u / segs);
        const long long from = (u - m * segs) * SEGMENT;
        const int2 mv = __ldcg(&w.moves[m]);
        const uint4 *s = reinterpret_cast<const uint4 *>(c.data + mv.x * bytes + from);
        uint4 *d = reinterpret_cast<uint4 *>(c.data + mv.y * bytes + from);
        const int n = static_cast<int>(min(static_cast<long long>(SEGMENT), bytes - from) / 16);
        uint4 v[SEGMENT / 16 / 256];
#pragma unroll
        for (int j = 0; j < SEGMENT / 16 / 256; ++j)
            if (static_cast<int>(threadIdx.x) + 256 * j < n) v[j] = s[threadIdx.x + 256 * j];
#pragma unroll
        for (int j = 0; j < SEGMENT / 16 / 256; ++j)
            if (static_cast<int>(threadIdx.x) + 256 * j < n) d[threadIdx.x + 256 * j] = v[j];
        if (from == 0)
            for (long long x = threadIdx.x; x < scales; x += 256) c.scale[mv.y * scales + x] = c.scale[mv.x * scales + x];
    }
}

__global__ void k_kv8_reset(const View c) {
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i < c.nPages) c.ref[i] = 0;
    if (i < c.nRow) c.len[i] = 0;
    if (i < static_cast<long long>(c.nRow) * c.maxPages) c.table[i] = -1;
}

// A launch whose CTAs start while the plan before it runs (it waits for the plan's end before it reads anything).
static int launch_after(void (*kern)(View, Work), int grid, cudaStream_t stream, const View &c, const Work &w) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, c, w) == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
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
    kv8::k_kv8_plan<<<1, kv8::PLAN_NT, 0, stream>>>(c, w, parent, advance, reserve);
    if (cudaGetLastError() != cudaSuccess) return GPT2_B200_ECUDA;
    if (reserve == 0) return GPT2_B200_OK;  // nothing is written next: no page is copied
    return kv8::launch_after(kv8::k_kv8_copy, ctx->num_sms * 4, stream, c, w);
}

int gpt2_kv8_compact_b200(const GPT2KV8Cache *kv, int *d_live, cudaStream_t stream) {
    if (kv8::check(kv) != GPT2_B200_OK || kv->work_bytes < kv8::work_layout(kv, kv->nHead, 1).bytes) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    const kv8::Work w = kv8::work_layout(kv, kv->nHead, 1);
    const kv8::View c = kv8::view(kv, ctx->status);
    kv8::k_kv8_compact_plan<<<1, kv8::PLAN_NT, 0, stream>>>(c, w, d_live);
    if (cudaGetLastError() != cudaSuccess) return GPT2_B200_ECUDA;
    return kv8::launch_after(kv8::k_kv8_compact_move, ctx->num_sms * 8, stream, c, w);
}

}  // extern "C"
