// beam_select.cu — the next beams out of beams x vocabulary candidates, in one launch and one pass.
//
// total(w, v) = score[w] + (x[w, v] - lse[w]), lse = m + log(sum exp(x - m)); a finished beam is the one candidate
// (w, eos) with its score. Within a beam totals fall as logits do, so a beam's W largest logits hold all
// of its candidates that matter: a row is read once, for the running maximum and sum and for its W largest logits.
// Reads 2 or 4 bytes per logit. The pass itself issues about 6 instructions per value; with lists, bounds and merges it is 24 for
// 64 items of 4 beams in fp16, whose warps wait for one another at the barriers more than for anything else (IPC 2.3, DRAM 14 %).
// Many fp32 rows are nearer HBM.
//
//   - Every warp streams its own part of a row through a ring of its own in shared memory (cp.async), so the main loop
//     has no CTA barrier and a warp has up to STAGES - 1 steps in flight. Rows are copied in aligned 16-byte
//     granules; lanes then take values by their index (neighbouring lanes neighbouring words, so that any alignment of
//     the row is read without bank conflicts), and equal rows get equal sums wherever they lie.
//   - The warp's W largest so far are a sorted list, lane j holding the j-th. A value is inserted if it reaches a
//     threshold that at least W values of the row reach: the list's last entry, or the smallest of the CTA's 8 warps' K-th
//     largest, K = ceil(W / 8); in the first step, without lists yet, of their lanes' maxima. About W ln(n / W) of a CTA's
//     n values are inserted; the others cost no more than their share of a maximum.
//   - Logits are compared as 64-bit keys: the value's orderable bits, then the inverted token, so equal logits go to the
//     lower token whatever the order of arrival.
//   - Sorted lists are merged by W rounds of a maximum over their heads, a lane per list: the warps' in a CTA, the CTAs' of
//     a row, and the beams' of an item, the last two by the item's last CTA to arrive (a counter that it re-arms).
//
// Measured over 50257 logits: 4 rows fp16 8.6 us (latency), 256 rows fp16 18.3 us (lists), 1024 rows fp32 47.9 us, 4.3 TB/s.
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
constexpr int NV = 16;          // values per lane and step
// Steps in a warp's ring: 4 KB and more in flight per warp, and for fp32 four CTAs per SM (with 4 stages three: a batch of 1024
// rows then takes three passes instead of two, 56 against 50 us).
template <typename T>
constexpr int stages() { return sizeof(T) == 4 ? 3 : 4; }
// A step's granules, and the one behind for rows that are not aligned.
template <typename T>
constexpr int stage_bytes() { return 32 * NV * static_cast<int>(sizeof(T)) + 16; }
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long key_t;

__host__ __device__ inline int max_chunks(int W) { return ROW_KEYS / W < MAX_CHUNKS ? ROW_KEYS / W : MAX_CHUNKS; }

// A row's part of the work area, of one size for every call, so that no call's lists lie where another's counters are: calls of
// any batch and width may share an area.
struct __align__(16) Record {
    key_t keys[ROW_KEYS];    // [chunks][W], sorted
    float2 ml[MAX_CHUNKS];   // [chunks]
    unsigned arrive, pad[3]; // the item's arrivals, in its first row's record; zero between calls
};

struct Params {
    int *token, *parent;
    float *new_score;
    int *new_done;
    const void *logits;
    long long ld;
    const float *score;
    const int *done;
    int W, V, eos, chunks, steps;  // steps per warp of a CTA
    Record *work;                  // [rows]
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
__device__ __forceinline__ key_t key_of(float x, unsigned n) { return lin::argmax_key(x + 0.0f, n); }  // -0 as 0: they are equal
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
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(unsigned o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// (m, l) over the warp, the same bits in every lane.
__device__ __forceinline__ void warp_ml(float &m, float &l) {
    const float mx = from_ordered(__reduce_max_sync(0xFFFFFFFFu, ordered(m)));
    l = m > -INFINITY ? l * ex2((m - mx) * LOG2E) : 0.0f;
    m = mx;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
}
// Merges n <= 64 descending lists of W keys (list i at a + i * W), one or two heads per lane; round j's
// winner goes to put(j, key, list). Stops when all are used up and returns how many were put.
template <typename Put>
__device__ __forceinline__ int merge_lists(const key_t *a, int n, int W, Put put) {
    const int lane = threadIdx.x & 31;
    int i0 = 0, i1 = 0;
    key_t k0 = lane < n ? a[lane * W] : 0, k1 = lane + 32 < n ? a[(lane + 32) * W] : 0;
#pragma unroll 1
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

// Two fp32 additions / multiplications as one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
template <typename T>
__global__ void __launch_bounds__(NT) k_beam_select(const Params p) {
    constexpr int EV = 16 / sizeof(T);       // values per granule
    constexpr int STEP = 32 * NV;            // values per warp and step
    constexpr int GPL = NV / EV;             // granules per lane and step
    constexpr int STAGE_BYTES = stage_bytes<T>(), STAGES = stages<T>();
    extern __shared__ __align__(16) uint8_t ring_all[];
    // behind the main loop the rings' memory holds the lists that are merged
    key_t (*lists)[ROW_KEYS] = reinterpret_cast<key_t (*)[ROW_KEYS]>(ring_all);
    key_t *totals = reinterpret_cast<key_t *>(ring_all + NWARP * ROW_KEYS * sizeof(key_t));  // [W][W]
    int *tokens = reinterpret_cast<int *>(totals + MAX_W * MAX_W);                           // [W][W]
    static_assert(NWARP * ROW_KEYS * 8 + MAX_W * MAX_W * 12 <= NWARP * stages<T>() * stage_bytes<T>(), "lists fit in the rings");
    __shared__ float red_m[NWARP], red_l[NWARP];
    __shared__ int is_last;
    __shared__ float kth[NWARP], kth2[NWARP];  // each warp's K-th largest value so far; its K2-th lane maximum
    __shared__ float cta_low;     // the smallest of them, as last seen
    __shared__ float s_score[MAX_W];
    __shared__ int s_done[MAX_W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = p.W, V = p.V;
    const int item = blockIdx.x / (W * p.chunks), rest = blockIdx.x - item * (W * p.chunks);
    const int w = rest / p.chunks, ch = rest - w * p.chunks;
    const long long row = static_cast<long long>(item) * W + w;
    const float my_score = p.score[row];
    const int my_done = p.done ? p.done[row] : 0;
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
            T part[EV];
#pragma unroll
            for (int j = 0; j < EV; ++j) part[j] = at + j >= 0 && at + j < V ? x[at + j] : static_cast<T>(-INFINITY);
            *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(part);
        }
    };
    auto load = [&](int s) {
        if (s < max(steps, 1)) {
            uint8_t *dst = ring + s % STAGES * STAGE_BYTES;
            const int base = begin + s * (NWARP * STEP) - shift;
            if (base >= 0 && base + STEP + EV <= V) {  // whole step inside the row
                const T *src = x + base + lane * EV;
#pragma unroll
                for (int q = 0; q < GPL; ++q) cp_async16(dst + (q * 32 + lane) * 16, src + q * 32 * EV);
                if (lane == 0) cp_async16(dst + 32 * GPL * 16, src + GPL * 32 * EV);
            } else {
                for (int q = 0; q < GPL; ++q) fetch(dst + (q * 32 + lane) * 16, base + (q * 32 + lane) * EV);
                if (lane == 0) fetch(dst + 32 * GPL * 16, base + 32 * GPL * EV);
            }
        }
        cp_async_commit();
    };
#pragma unroll 1
    for (int s = 0; s < STAGES - 1; ++s) load(s);  // before the beam's state is there: most beams are alive
    const bool alive = my_score > -INFINITY && !my_done;
    if (!alive) cp_async_wait<0>();
    if (alive) {
        float m = -INFINITY, l = 0.0f;
        key_t mine = 0, worst = 0;  // the j-th largest key in lane j; the W-th
        float thr = -INFINITY, low = -INFINITY;
        bool bad = false;
        // The CTA's warps that have values; K values of each are W in all, and K2 of half of them.
        const int active = max(1, min(NWARP, (V - ch * p.steps * NWARP * STEP + STEP - 1) / STEP));
        const int K = (W + active - 1) / active, K2 = (W + (active + 1) / 2 - 1) / ((active + 1) / 2);
        auto row_low = [&](int i) {
            const float x = i < active ? *const_cast<volatile float *>(&kth[i & (NWARP - 1)]) : INFINITY;
            return from_ordered(__reduce_min_sync(0xFFFFFFFFu, ordered(x)));
        };
        // The count-th largest of the lanes' x, and the at-th on the way (by lane 0).
        auto kth_of_warp = [&](float x, int count, int at, float &kept) {
            unsigned o = ordered(x), mx = 0;
#pragma unroll 1
            for (int j = 1; j <= count; ++j) {
                mx = __reduce_max_sync(0xFFFFFFFFu, o);
                if (lane == __ffs(__ballot_sync(0xFFFFFFFFu, o == mx)) - 1) o = 0;
                if (j == at && lane == 0) kept = from_ordered(mx);
            }
            return from_ordered(mx);
        };
        if (tid == 0) cta_low = -INFINITY;  // before the barrier of step 0
        for (int s = 0; s < max(steps, 1); ++s) {  // a warp without values has one step of -inf, for the barrier in it
            cp_async_wait<STAGES - 2>();
            __syncwarp();  // every lane's copies of step s are there, and all are done with step s - 1
            load(s + STAGES - 1);
            // value i of lane: fp32: 32 i + lane; fp16: 64 (i / 2) + 2 lane + i % 2
            const uint8_t *src = ring + s % STAGES * STAGE_BYTES + (cut & ~3u) + lane * 4;
            float2 v[NV / 2];
            float top;
            if (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < NV / 2; ++i)
                    v[i] = make_float2(*reinterpret_cast<const float *>(src + 256 * i), *reinterpret_cast<const float *>(src + 256 * i + 128));
                top = max_nan(v[0].x, v[0].y);
#pragma unroll
                for (int i = 1; i < NV / 2; ++i) top = max_nan(top, max_nan(v[i].x, v[i].y));
            } else {
                __half2 h[NV / 2];
#pragma unroll
                for (int i = 0; i < NV / 2; ++i) {
                    uint32_t u = *reinterpret_cast<const uint32_t *>(src + 128 * i);
                    if (cut & 2) u = __funnelshift_r(u, *reinterpret_cast<const uint32_t *>(src + 128 * i + 4), 16);
                    h[i] = *reinterpret_cast<const __half2 *>(&u);
                    v[i] = __half22float2(h[i]);
                }
#pragma unroll
                for (int o = NV / 4; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < o; ++i) h[i] = __hmax2_nan(h[i], h[i + o]);
                const float2 f = __half22float2(h[0]);
                top = max_nan(f.x, f.y);
            }
            if (!(top < INFINITY)) {  // NaN and +inf count as masked
                bad = true;
                top = -INFINITY;
#pragma unroll
                for (int i = 0; i < NV / 2; ++i) {
                    v[i].x = v[i].x < INFINITY ? v[i].x : -INFINITY;
                    v[i].y = v[i].y < INFINITY ? v[i].y : -INFINITY;
                    top = fmaxf(top, fmaxf(v[i].x, v[i].y));
                }
            }
            if (top > m) {
                l *= ex2((m - top) * LOG2E);
                m = top;
            }
            if (m > -INFINITY) {  // m subtracted first: exact near m, where it counts
                const float2 mm = make_float2(-m, -m), ll = make_float2(LOG2E, LOG2E);
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < NV / 2; ++i) {
                    const float2 e = mul2(add2(v[i], mm), ll);
                    sum = add2(sum, make_float2(ex2(e.x), ex2(e.y)));
                }
                l += sum.x + sum.y;
            }
            if (s == 0) {
                const float kb = kth_of_warp(top, K2, K, kth[warp]);
                if (lane == 0) kth2[warp] = kb;
                __syncthreads();
                low = row_low(lane);
                // the (A + 1) / 2-th largest of the warps' K2-th: a warp at the row's end, with few values, does not lower it
                float unused;
                low = fmaxf(low, kth_of_warp(lane < active ? kth2[lane & (NWARP - 1)] : -INFINITY, (active + 1) / 2, 0, unused));
            } else {
                low = *const_cast<volatile float *>(&cta_low);
            }
            thr = fmaxf(thr, low);
            // Each lane with such a value: 16 lanes look at its values again, in the ring, and those that reach the
            // threshold are inserted, which raises it for the lanes that are left.
            unsigned from = __ballot_sync(0xFFFFFFFFu, top >= thr && top > -INFINITY);
            if (!from) continue;
            do {
                const int who = __ffs(from) - 1;
                from &= from - 1;
                const unsigned at = sizeof(T) == 4 ? 32 * lane + who : 64 * (lane >> 1) + 2 * who + (lane & 1);
                key_t k = 0;
                if (lane < NV) {
                    const float y = static_cast<float>(*reinterpret_cast<const T *>(ring + s % STAGES * STAGE_BYTES + cut + at * sizeof(T)));
                    if (y >= thr && y > -INFINITY && y < INFINITY) k = key_of(y, begin + s * (NWARP * STEP) + at);
                }
#pragma unroll 1
                for (unsigned todo = __ballot_sync(0xFFFFFFFFu, k > worst); todo; todo &= todo - 1) {
                    const key_t in_key = __shfl_sync(0xFFFFFFFFu, k, __ffs(todo) - 1);
                    const int rank = __popc(__ballot_sync(0xFFFFFFFFu, mine > in_key));
                    const key_t up = __shfl_up_sync(0xFFFFFFFFu, mine, 1);
                    if (lane >= rank && lane < W) mine = lane == rank ? in_key : up;
                }
                worst = __shfl_sync(0xFFFFFFFFu, mine, W - 1);
                if (worst) thr = fmaxf(thr, key_value(worst));
                from &= __ballot_sync(0xFFFFFFFFu, top >= thr);
            } while (from);
            // the CTA's bound; two warps may write it at once, either value holds
            if (lane == K - 1 && mine) *const_cast<volatile float *>(&kth[warp]) = fmaxf(kth[warp], key_value(mine));
            __syncwarp();
            low = row_low(lane);
            if (lane == 0 && low > *const_cast<volatile float *>(&cta_low)) *const_cast<volatile float *>(&cta_low) = low;
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
        Record *const rec = p.work + row;
        if (warp == 0) {
            key_t *out = rec->keys + ch * W;
            const int n = merge_lists(lists[0], NWARP, W, [&](int j, key_t k, int) { out[j] = k; });
            if (lane >= n && lane < W) out[lane] = 0;
        } else if (warp == 1) {
            m = lane < NWARP ? red_m[lane] : -INFINITY;
            l = lane < NWARP ? red_l[lane] : 0.0f;
            warp_ml(m, l);
            if (lane == 0) rec->ml[ch] = make_float2(m, l);
        }
    }
    // the last CTA of the item goes on
    const int first_row = item * W;
    if (tid < W) {
        s_score[tid] = p.score[first_row + tid];
        s_done[tid] = p.done ? p.done[first_row + tid] : 0;
    }
    __syncthreads();
    if (tid == 0) {
        unsigned *const arrive = &p.work[first_row].arrive;
        const unsigned seen = kv8::arrive_add(arrive);
        is_last = seen == static_cast<unsigned>(W * p.chunks - 1);
        if (is_last) *arrive = 0;
    }
    __syncthreads();
    if (!is_last) return;
    for (int i = tid; i < W * W; i += NT) totals[i] = 0;
    __syncthreads();
    // a warp per beam: lse, the beam's W best logits, their totals
    for (int b = warp; b < W; b += NWARP) {
        const float sc = s_score[b];
        if (!(sc > -INFINITY)) continue;
        if (s_done[b]) {
            if (lane == 0) {
                totals[b * W] = key_of(sc, static_cast<unsigned>(b * W));
                tokens[b * W] = max(p.eos, 0);
            }
            continue;
        }
        const Record *const rec = p.work + first_row + b;
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < p.chunks; i += 32) {
            const float2 z = __ldcg(&rec->ml[i]);
            merge_ml(m, l, z.x, z.y);
        }
        for (int i = lane; i < p.chunks * W; i += 32) lists[warp][i] = __ldcg(&rec->keys[i]);
        warp_ml(m, l);
        __syncwarp();
        const float lse = m + logf(l);
        auto candidate = [&](int j, key_t k, int) {
            totals[b * W + j] = key_of(sc + (key_value(k) - lse), static_cast<unsigned>(b * W + j));
            tokens[b * W + j] = lin::argmax_key_index(k);
        };
        if (p.chunks > 1) merge_lists(lists[warp], p.chunks, W, candidate);
        else if (lane < W && lists[warp][lane]) candidate(lane, lists[warp][lane], 0);
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

template <typename T>
static int launch(Params p, int B, int num_sms, bool *attr_done, cudaStream_t stream) {
    constexpr int STEP = 32 * NV;
    constexpr int SMEM = NWARP * stages<T>() * stage_bytes<T>();
    const long long rows = static_cast<long long>(B) * p.W;
    // CTAs of a row. One pass of all resident CTAs costs a CTA's steps and about as much as FIXED steps to start and to
    // merge; the number of CTAs per row that makes passes x cost least is taken. Few rows so come down to one step per warp,
    // and many rows do not leave a last pass with a few CTAs.
    constexpr long long FIXED = 3;
    const long long slots = static_cast<long long>(num_sms) * (228 * 1024 / (SMEM + 2048));
    const long long groups = (p.V + NWARP * STEP - 1) / (NWARP * STEP);  // steps of a CTA that had the row to itself
    long long best = 0;
    for (long long c = 1; c <= std::min<long long>(groups, max_chunks(p.W)); ++c) {
        const long long steps = (groups + c - 1) / c, used = (groups + steps - 1) / steps;
        const long long cost = (rows * used + slots - 1) / slots * (steps + FIXED);
        if (used == c && (!best || cost < best)) {
            best = cost;
            p.chunks = static_cast<int>(c);
            p.steps = static_cast<int>(steps);
        }
    }
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
    return static_cast<size_t>(B) * W * sizeof(beam::Record);
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
    if (work_bytes < gpt2_beam_work_bytes_b200(B, W)) return GPT2_B200_EINVAL;
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
    p.work = static_cast<beam::Record *>(work);
    p.status = ctx->status;
    return type == GPT2_BEAM_HALF ? beam::launch<__half>(p, B, ctx->num_sms, &ctx->beam_attr_done[0], stream)
                                  : beam::launch<float>(p, B, ctx->num_sms, &ctx->beam_attr_done[1], stream);
}
