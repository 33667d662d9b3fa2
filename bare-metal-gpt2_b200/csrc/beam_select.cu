// beam_select.cu — the next beams out of beams x vocabulary candidates, in one launch and one pass.
//
// total(w, v) = score[w] + (x[w, v] - lse[w]), lse = m + log(sum exp(x - m)); a finished beam is the one candidate
// (w, eos) with its score. Within a beam totals fall as logits do, so a beam's W largest logits hold all
// of its candidates that matter: a row is read once, for the running maximum and sum and for its W largest logits.
// Bound by reading the logits from HBM (2 or 4 bytes each; about 8 instructions per value).
//
//   - Every warp streams its own part of a row through a ring of its own in shared memory (cp.async), so the main loop
//     has no CTA barrier and a warp has up to STAGES - 1 steps in flight. Lanes own values by their index, whatever the
//     row's alignment: equal rows get equal sums. A row that does not start on a 16-byte boundary is copied in aligned
//     granules and a lane's values are cut out of two neighbouring ones.
//   - The warp's W largest so far are a sorted list, lane j holding the j-th; its last entry is the threshold that a value
//     must pass to be inserted (about W ln(n / W) of n values do). The first step starts from a threshold that at
//     least W values reach: the W-th largest of the lanes' maxima.
//   - Logits are compared as 64-bit keys: the value's orderable bits, then the inverted token, so equal logits go to the
//     lower token whatever the order of arrival.
//   - Sorted lists are merged by W rounds of a maximum over their heads, a lane per list: the warps' in a CTA, the CTAs' of
//     a row, and the beams' of an item, the last two by the item's last CTA to arrive (a counter that it re-arms).
#include <algorithm>

#include "kv8.cuh"
#include "linear.cuh"
#include "ptx.cuh"

namespace b200 {
namespace beam {

constexpr int MAX_W = 32;
constexpr int NWARP = 8, NT = 32 * NWARP;
constexpr int MAX_CHUNKS = 64;  // CTAs of a row: two list heads per lane
constexpr int ROW_KEYS = 256;   // CTAs x W of a row, at most
constexpr int VPT = 2;          // 16-byte granules per lane and step
constexpr int STAGES = 6;
constexpr int STAGE_BYTES = (32 * VPT + 1) * 16;  // and the granule behind, for rows that are not aligned
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long key_t;

__host__ __device__ inline int max_chunks(int W) { return ROW_KEYS / W < MAX_CHUNKS ? ROW_KEYS / W : MAX_CHUNKS; }

struct Params {
    int *token, *parent;
    float *new_score;
    int *new_done;
    const void *logits;
    long long ld;
    const float *score;
    const int *done;
    int W, V, eos, chunks, steps;  // steps per warp of a CTA
    key_t *keys;                   // [rows][chunks][W], sorted
    float2 *ml;                    // [rows][chunks]
    unsigned *arrive;              // [items]
    unsigned *status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float key_value(key_t k) {
    const unsigned o = static_cast<unsigned>(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ key_t warp_max(key_t k) {
    const unsigned hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(k >> 32));
    const unsigned lo = __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned>(k >> 32) == hi ? static_cast<unsigned>(k) : 0u);
    return (static_cast<key_t>(hi) << 32) | lo;
}
__device__ __forceinline__ void merge_ml(float &m, float &l, float m2, float l2) {
    const float mx = fmaxf(m, m2);
    if (mx == -INFINITY) return;
    l = l * ex2((m - mx) * LOG2E) + l2 * ex2((m2 - mx) * LOG2E);
    m = mx;
}
// (m, l) over the warp, the same bits in every lane.
__device__ __forceinline__ void warp_ml(float &m, float &l) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, o);
        const bool upper = threadIdx.x & o;  // both sides add in the same order
        float a = upper ? m2 : m, b = upper ? l2 : l;
        merge_ml(a, b, upper ? m : m2, upper ? l : l2);
        m = a;
        l = b;
    }
}
// Merges n <= 64 descending lists of W keys (list i at a + i * W), one or two heads per lane; round j's
// winner goes to put(j, key, list). Stops when all are used up and returns how many were put.
template <typename Put>
__device__ __forceinline__ int merge_lists(const key_t *a, int n, int W, Put put) {
    const int lane = threadIdx.x & 31;
    int i0 = 0, i1 = 0;
    key_t k0 = lane < n ? a[lane * W] : 0, k1 = lane + 32 < n ? a[(lane + 32) * W] : 0;
    for (int j = 0; j < W; ++j) {
        const key_t top = warp_max(max(k0, k1));
        if (!top) return j;
        if (k0 == top) {  // keys are distinct: one lane pops
            put(j, top, lane);
            k0 = ++i0 < W ? a[lane * W + i0] : 0;
        } else if (k1 == top) {
            put(j, top, lane + 32);
            k1 = ++i1 < W ? a[(lane + 32) * W + i1] : 0;
        }
    }
    return W;
}
__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
__device__ __forceinline__ void unpack(const uint32_t (&w)[4], float *v);
template <>
__device__ __forceinline__ void unpack<float>(const uint32_t (&w)[4], float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint32_t (&w)[4], float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) k_beam_select(const Params p) {
    constexpr int EV = 16 / sizeof(T);    // values per granule
    constexpr int STEP = 32 * VPT * EV;   // values per warp and step
    constexpr int NV = VPT * EV;          // values per lane and step
    extern __shared__ __align__(16) uint8_t ring_all[];
    // behind the main loop the rings' memory holds the lists that are merged
    key_t (*lists)[ROW_KEYS] = reinterpret_cast<key_t (*)[ROW_KEYS]>(ring_all);
    key_t *totals = reinterpret_cast<key_t *>(ring_all + NWARP * ROW_KEYS * sizeof(key_t));  // [W][W]
    int *tokens = reinterpret_cast<int *>(totals + MAX_W * MAX_W);                           // [W][W]
    static_assert(NWARP * ROW_KEYS * 8 + MAX_W * MAX_W * 12 <= NWARP * STAGES * STAGE_BYTES, "lists fit in the rings");
    __shared__ float red_m[NWARP], red_l[NWARP];
    __shared__ int is_last;
    __shared__ float s_score[MAX_W];
    __shared__ int s_done[MAX_W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = p.W, V = p.V;
    const int item = blockIdx.x / (W * p.chunks), rest = blockIdx.x - item * (W * p.chunks);
    const int w = rest / p.chunks, ch = rest - w * p.chunks;
    const long long row = static_cast<long long>(item) * W + w;
    const bool alive = p.score[row] > -INFINITY && !(p.done && p.done[row]);
    if (alive) {
        const T *x = static_cast<const T *>(p.logits) + row * p.ld;
        const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        const unsigned cut = shift * sizeof(T);
        uint8_t *ring = ring_all + warp * STAGES * STAGE_BYTES;
        const int begin = (ch * p.steps * NWARP + warp) * STEP;  // step s: values begin + s * NWARP * STEP ..
        int steps = begin < V ? min(p.steps, (V - begin + NWARP * STEP - 1) / (NWARP * STEP)) : 0;
        // Granule g of a step holds values base + g * EV - shift ..; outside the row they are -inf. One that
        // reaches over the row's ends is read value by value.
        auto fetch = [&](uint8_t *dst, int at) {
            if (at >= 0 && at + EV <= V) {
                cp_async16(dst, x + at);
            } else {
#pragma unroll
                for (int j = 0; j < EV; ++j)
                    reinterpret_cast<T *>(dst)[j] = at + j >= 0 && at + j < V ? x[at + j] : static_cast<T>(-INFINITY);
            }
        };
        auto load = [&](int s) {
            if (s < steps) {
                uint8_t *dst = ring + s % STAGES * STAGE_BYTES;
                const int base = begin + s * (NWARP * STEP) - shift;
#pragma unroll
                for (int q = 0; q < VPT; ++q) fetch(dst + (q * 32 + lane) * 16, base + (q * 32 + lane) * EV);
                if (cut && lane == 0) fetch(dst + 32 * VPT * 16, base + 32 * VPT * EV);
            }
            cp_async_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) load(s);
        float m = -INFINITY, l = 0.0f;
        key_t mine = 0, worst = 0;  // the j-th largest key in lane j; the W-th
        float thr = -INFINITY;
        bool bad = false;
        for (int s = 0; s < steps; ++s) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of step s are there, and all are done with step s - 1
            load(s + STAGES - 1);
            const uint4 *src = reinterpret_cast<const uint4 *>(ring + s % STAGES * STAGE_BYTES);
            float v[NV];
#pragma unroll
            for (int q = 0; q < VPT; ++q) {
                const uint4 a = src[q * 32 + lane];
                uint32_t o[4] = {a.x, a.y, a.z, a.w};
                if (cut) {
                    const uint4 b = src[q * 32 + lane + 1];
                    uint32_t c[5];
                    switch (cut >> 2) {
                        case 0: c[0] = a.x, c[1] = a.y, c[2] = a.z, c[3] = a.w, c[4] = b.x; break;
                        case 1: c[0] = a.y, c[1] = a.z, c[2] = a.w, c[3] = b.x, c[4] = b.y; break;
                        case 2: c[0] = a.z, c[1] = a.w, c[2] = b.x, c[3] = b.y, c[4] = b.z; break;
                        default: c[0] = a.w, c[1] = b.x, c[2] = b.y, c[3] = b.z, c[4] = b.w; break;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(c[i], c[i + 1], (cut & 2) * 8);
                }
                unpack<T>(o, v + q * EV);
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < NV; ++i) top = max_nan(top, v[i]);
            if (!(top < INFINITY)) {  // NaN and +inf count as masked
                bad = true;
                top = -INFINITY;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    v[i] = v[i] < INFINITY ? v[i] : -INFINITY;
                    top = fmaxf(top, v[i]);
                }
            }
            if (top > m) {
                l *= ex2((m - top) * LOG2E);
                m = top;
            }
            if (m > -INFINITY) {
#pragma unroll
                for (int i = 0; i < NV; ++i) l += ex2((v[i] - m) * LOG2E);  // m subtracted first: exact near m, where it counts
            }
            if (s == 0) {  // the W-th largest of the 32 lane maxima: no W values are lost below it
                int rank = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float u = __shfl_sync(0xFFFFFFFFu, top, i);
                    rank += u > top || (u == top && i < lane);
                }
                const unsigned who = __ballot_sync(0xFFFFFFFFu, rank == W - 1);
                thr = __shfl_sync(0xFFFFFFFFu, top, __ffs(who) - 1);
            }
            if (!__any_sync(0xFFFFFFFFu, top >= thr && top > -INFINITY)) continue;
            const unsigned first = begin + s * (NWARP * STEP) + lane * EV;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const bool in = v[i] >= thr && v[i] > -INFINITY;
                unsigned todo = __ballot_sync(0xFFFFFFFFu, in);
                if (!todo) continue;
                const key_t k = lin::argmax_key(v[i], first + i / EV * 32 * EV + i % EV);
                todo = __ballot_sync(0xFFFFFFFFu, in && k > worst);
                while (todo) {
                    const int from = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const key_t in_key = __shfl_sync(0xFFFFFFFFu, k, from);
                    const int rank = __popc(__ballot_sync(0xFFFFFFFFu, mine > in_key));
                    const key_t up = __shfl_up_sync(0xFFFFFFFFu, mine, 1);
                    if (lane >= rank && lane < W) mine = lane == rank ? in_key : up;
                }
                worst = __shfl_sync(0xFFFFFFFFu, mine, W - 1);
                if (worst) thr = key_value(worst);
            }
        }
        warp_ml(m, l);
        if (lane == 0) {
            red_m[warp] = m;
            red_l[warp] = l;
        }
        __syncthreads();  // every warp is through its ring
        if (lane < W) lists[0][warp * W + lane] = mine;
        if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.status, ST_BEAM_LOGIT);
        __syncthreads();
        const long long at = row * p.chunks + ch;
        if (warp == 0) {
            key_t *out = p.keys + at * W;
            const int n = merge_lists(lists[0], NWARP, W, [&](int j, key_t k, int) { out[j] = k; });
            if (lane >= n && lane < W) out[lane] = 0;
        } else if (warp == 1) {
            m = lane < NWARP ? red_m[lane] : -INFINITY;
            l = lane < NWARP ? red_l[lane] : 0.0f;
            warp_ml(m, l);
            if (lane == 0) p.ml[at] = make_float2(m, l);
        }
    }
    // the last CTA of the item goes on
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const unsigned seen = atomicAdd(&p.arrive[item], 1u);
        is_last = seen == static_cast<unsigned>(W * p.chunks - 1);
        if (is_last) p.arrive[item] = 0;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    const int first_row = item * W;
    if (tid < W) {
        s_score[tid] = p.score[first_row + tid];
        s_done[tid] = p.done ? p.done[first_row + tid] : 0;
    }
    for (int i = tid; i < W * W; i += NT) totals[i] = 0;
    __syncthreads();
    // a warp per beam: lse, the beam's W best logits, their totals
    for (int b = warp; b < W; b += NWARP) {
        const float sc = s_score[b];
        if (!(sc > -INFINITY)) continue;
        if (s_done[b]) {
            if (lane == 0) {
                totals[b * W] = lin::argmax_key(sc, static_cast<unsigned>(b * W));
                tokens[b * W] = max(p.eos, 0);
            }
            continue;
        }
        const long long at = static_cast<long long>(first_row + b) * p.chunks;
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < p.chunks; i += 32) {
            const float2 z = __ldcg(&p.ml[at + i]);
            merge_ml(m, l, z.x, z.y);
        }
        for (int i = lane; i < p.chunks * W; i += 32) lists[warp][i] = __ldcg(&p.keys[at * W + i]);
        warp_ml(m, l);
        __syncwarp();
        const float lse = m + logf(l);
        merge_lists(lists[warp], p.chunks, W, [&](int j, key_t k, int) {
            totals[b * W + j] = lin::argmax_key(sc + (key_value(k) - lse), static_cast<unsigned>(b * W + j));
            tokens[b * W + j] = lin::argmax_key_index(k);
        });
        __syncwarp();
    }
    __syncthreads();
    if (warp != 0) return;
    // a beam's totals fall with its logits (rounding keeps the order; equal ones by rank): sorted lists again
    const int n = merge_lists(totals, W, W, [&](int j, key_t k, int b) {
        const int out = first_row + j, token = tokens[lin::argmax_key_index(k)];
        p.token[out] = token;
        p.parent[out] = first_row + b;
        p.new_score[out] = key_value(k);
        if (p.new_done) p.new_done[out] = s_done[b] || token == p.eos;
    });
    if (lane >= n && lane < W) {  // fewer candidates than beams: the rest are dead
        const int out = first_row + lane;
        p.token[out] = max(p.eos, 0);
        p.parent[out] = out;
        p.new_score[out] = -INFINITY;
        if (p.new_done) p.new_done[out] = 1;
    }
}

struct Layout {
    size_t o_keys, o_ml, bytes;
};
static Layout layout(int B, int W) {
    auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    const size_t rows = static_cast<size_t>(B) * W, ch = static_cast<size_t>(max_chunks(W));
    Layout y;
    y.o_keys = up(B * sizeof(unsigned));
    y.o_ml = y.o_keys + up(rows * ch * W * sizeof(key_t));
    y.bytes = y.o_ml + up(rows * ch * sizeof(float2));
    return y;
}

template <typename T>
static int launch(Params p, int B, int num_sms, bool *attr_done, cudaStream_t stream) {
    constexpr int STEP = 32 * VPT * (16 / static_cast<int>(sizeof(T)));
    constexpr int SMEM = NWARP * STAGES * STAGE_BYTES;
    const long long rows = static_cast<long long>(B) * p.W;
    // CTAs of a row: about four per SM in all; down to one step per warp when rows are few (bound by the latency
    // of one CTA), the whole row when they are many.
    const long long groups = (p.V + NWARP * STEP - 1) / (NWARP * STEP);  // steps of a CTA that had the row to itself
    long long chunks = (4ll * num_sms + rows - 1) / rows;
    chunks = std::min<long long>({chunks, groups, max_chunks(p.W)});
    p.steps = static_cast<int>((groups + chunks - 1) / chunks);
    p.chunks = static_cast<int>((groups + p.steps - 1) / p.steps);
    const long long grid = rows * p.chunks;
    if (grid > 0x7FFFFFFFll) return GPT2_B200_EINVAL;
    if (!*attr_done) {
        RelaxedCapture relaxed;
        if (cudaFuncSetAttribute(k_beam_select<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess)
            return GPT2_B200_ECUDA;
        *attr_done = true;
    }
    k_beam_select<T><<<static_cast<unsigned>(grid), NT, SMEM, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // namespace beam
}  // namespace b200

using namespace b200;

extern "C" size_t gpt2_beam_work_bytes_b200(int B, int W) {
    if (B < 1 || W < 1 || W > beam::MAX_W) return 0;
    return beam::layout(B, W).bytes;
}

extern "C" int gpt2_beam_select_b200(int *token, int *parent, float *new_score, int *new_done, const void *logits,
                                     int type, long long ld, const float *score, const int *done, int B, int W, int V,
                                     int eos, void *work, size_t work_bytes, cudaStream_t stream) {
    if (!token || !parent || !new_score || !logits || !score || !kv8::aligned(work) || B < 0 || W < 1 || W > beam::MAX_W ||
        V < 1 || V >= 1 << 30 || ld < V || eos < -1 || eos >= V || static_cast<long long>(B) * W > 0x7FFFFFFFll ||
        (type != GPT2_BEAM_HALF && type != GPT2_BEAM_FLOAT) ||
        (reinterpret_cast<uintptr_t>(logits) & (type == GPT2_BEAM_HALF ? 1 : 3)))
        return GPT2_B200_EINVAL;
    if (B == 0) return GPT2_B200_OK;
    const beam::Layout y = beam::layout(B, W);
    if (work_bytes < y.bytes) return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    beam::Params p;
    p.token = token;
    p.parent = parent;
    p.new_score = new_score;
    p.new_done = new_done;
    p.logits = logits;
    p.ld = ld;
    p.score = score;
    p.done = done;
    p.W = W;
    p.V = V;
    p.eos = eos;
    p.arrive = static_cast<unsigned *>(work);
    p.keys = reinterpret_cast<beam::key_t *>(static_cast<char *>(work) + y.o_keys);
    p.ml = reinterpret_cast<float2 *>(static_cast<char *>(work) + y.o_ml);
    p.status = ctx->status;
    return type == GPT2_BEAM_HALF ? beam::launch<__half>(p, B, ctx->num_sms, &ctx->beam_attr_done[0], stream)
                                  : beam::launch<float>(p, B, ctx->num_sms, &ctx->beam_attr_done[1], stream);
}
