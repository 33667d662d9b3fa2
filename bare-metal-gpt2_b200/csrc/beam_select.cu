// beam_select.cu — the next beams out of beams x vocabulary candidates, in one launch and one pass.
//
// total(w, v) = score[w] + (x[w, v] - lse[w]), lse = m + log(sum exp(x - m)); a finished beam is the one candidate
// (w, eos) with its score. Within a beam totals fall as logits do, so a beam's W largest logits hold all
// of its candidates that matter: a row is read once, for the running maximum and sum and for its W largest logits.
// Bound by reading the logits from HBM (2 or 4 bytes each, one exponential per value).
//
//   - A CTA takes a chunk of a row, tile by tile, a tile in registers (16-byte loads, also of rows that are
//     not aligned). Each thread keeps its own (m, l).
//   - The W largest of a tile without a sort: of G >= W disjoint groups of threads each has a maximum, so the smallest of
//     the G maxima is at most the W-th largest value. Values at least that (about G ln G of them, 22 for 8) go to a
//     list, and a value's rank is the number of list entries before it. A list that overflows (many equal
//     values) is replaced by W rounds of a maximum below the last one.
//   - Logits are compared as 64-bit keys: the value's orderable bits, then the inverted token, so equal logits go to the
//     lower token whatever the order of arrival.
//   - The last CTA of an item to arrive (a counter that it re-arms) merges its rows: a key's rank among the sorted
//     lists of a row's chunks is found by binary search; then the W x W totals the same way, equal
//     totals by the lower beam.
#include <algorithm>

#include "kv8.cuh"
#include "linear.cuh"

namespace b200 {
namespace beam {

constexpr int MAX_W = 32;
constexpr int NT = 256, NWARP = NT / 32;
constexpr int MAX_CHUNKS = 64;    // chunks of a row
constexpr int ROW_KEYS = 256;     // chunks x W of a row, at most
constexpr int LIST = 1024;        // candidates of a tile
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
    int W, V, eos, chunks, chunk;  // chunk: values per CTA
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
__device__ __forceinline__ float key_value(key_t k) {
    const unsigned o = static_cast<unsigned>(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// Entries of the descending list a[0..n) above k.
__device__ __forceinline__ int above(const key_t *a, int n, key_t k) {
    int lo = 0;
    while (n > 0) {
        const int half = n >> 1;
        if (a[lo + half] > k) {
            lo += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return lo;
}
__device__ __forceinline__ void merge_ml(float &m, float &l, float m2, float l2) {
    const float mx = fmaxf(m, m2);
    if (mx == -INFINITY) return;
    l = l * ex2((m - mx) * LOG2E) + l2 * ex2((m2 - mx) * LOG2E);
    m = mx;
}

// VPT 16-byte vectors per thread and tile.
template <typename T, int VPT>
__global__ void __launch_bounds__(NT) k_beam_select(const Params p) {
    constexpr int EV = 16 / sizeof(T);  // values per vector
    constexpr int TILE = NT * VPT * EV;
    __shared__ key_t list[LIST];
    __shared__ key_t run[2][MAX_W];
    __shared__ float gmax[NWARP * 4];
    __shared__ float red_m[NWARP], red_l[NWARP];
    __shared__ key_t red_k[NWARP];
    __shared__ int count, is_last;
    __shared__ key_t rowbuf[NWARP][ROW_KEYS];
    __shared__ float s_score[MAX_W];
    __shared__ int s_done[MAX_W];
    __shared__ key_t final_keys[MAX_W * MAX_W];
    __shared__ int final_token[MAX_W * MAX_W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = p.W, V = p.V;
    const int item = blockIdx.x / (W * p.chunks), rest = blockIdx.x - item * (W * p.chunks);
    const int w = rest / p.chunks, ch = rest - w * p.chunks;
    const long long row = static_cast<long long>(item) * W + w;
    const bool alive = p.score[row] > -INFINITY && !(p.done && p.done[row]);
    if (alive) {
        const T *x = static_cast<const T *>(p.logits) + row * p.ld;
        // Thread and tile own values by their index, whatever the row's alignment: equal rows get equal sums. A row that
        // starts `shift` values behind a 16-byte boundary is read in aligned granules, and a thread's vector is cut out
        // of two neighbouring ones (the second comes from L1). Granules that reach over the row's ends are read value by value.
        const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        const unsigned cut = shift * sizeof(T);
        const int begin = ch * p.chunk, end = min(begin + p.chunk, V);
        auto granule = [&](int at) {  // values at .. at + EV - 1, -inf outside the row
            uint4 g;
            if (at >= 0 && at + EV <= V) {
                asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(g.x), "=r"(g.y), "=r"(g.z), "=r"(g.w) : "l"(x + at));
            } else {
                T part[EV];
#pragma unroll
                for (int j = 0; j < EV; ++j) part[j] = at + j >= 0 && at + j < V ? x[at + j] : static_cast<T>(-INFINITY);
                g = *reinterpret_cast<uint4 *>(part);
            }
            return g;
        };
        float m = -INFINITY, l = 0.0f;
        bool bad = false;
        if (tid < 2 * MAX_W) run[tid / MAX_W][tid % MAX_W] = 0;
        int cur = 0;
        for (int base = begin; base < end; base += TILE) {
            float v[VPT][EV];
            uint4 raw[VPT], next[VPT];
#pragma unroll
            for (int q = 0; q < VPT; ++q) {
                const int at = base + (q * NT + tid) * EV;
                raw[q] = granule(at - shift);
                if (cut) next[q] = granule(at - shift + EV);
            }
            if (cut) {
#pragma unroll
                for (int q = 0; q < VPT; ++q) {
                    const uint4 &y = raw[q], &z = next[q];
                    uint32_t s[5];
                    switch (cut >> 2) {
                        case 0: s[0] = y.x, s[1] = y.y, s[2] = y.z, s[3] = y.w, s[4] = z.x; break;
                        case 1: s[0] = y.y, s[1] = y.z, s[2] = y.w, s[3] = z.x, s[4] = z.y; break;
                        case 2: s[0] = y.z, s[1] = y.w, s[2] = z.x, s[3] = z.y, s[4] = z.z; break;
                        default: s[0] = y.w, s[1] = z.x, s[2] = z.y, s[3] = z.z, s[4] = z.w; break;
                    }
                    const unsigned bits = (cut & 2) * 8;
                    raw[q] = make_uint4(__funnelshift_r(s[0], s[1], bits), __funnelshift_r(s[1], s[2], bits),
                                        __funnelshift_r(s[2], s[3], bits), __funnelshift_r(s[3], s[4], bits));
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < VPT; ++q) {
                const T *e = reinterpret_cast<const T *>(&raw[q]);
#pragma unroll
                for (int j = 0; j < EV; ++j) {
                    const float y = static_cast<float>(e[j]);
                    v[q][j] = y < INFINITY ? y : -INFINITY;  // NaN and +inf count as masked
                    bad |= !(y < INFINITY);
                    top = fmaxf(top, v[q][j]);
                }
            }
            if (top > m) {
                l *= ex2((m - top) * LOG2E);
                m = top;
            }
            if (m > -INFINITY) {
#pragma unroll
                for (int q = 0; q < VPT; ++q)
#pragma unroll
                    for (int j = 0; j < EV; ++j) l += ex2((v[q][j] - m) * LOG2E);  // m subtracted first: exact near m, where it counts
            }
            // the group maxima: groups of 32 threads (W <= 8), of 16 or of 8
            float gm = top;
            const int per = W <= 8 ? 32 : W <= 16 ? 16 : 8;
            for (int o = 1; o < per; o <<= 1) gm = fmaxf(gm, __shfl_xor_sync(0xFFFFFFFFu, gm, o));
            if (tid % per == 0) gmax[tid / per] = gm;
            if (tid == 0) count = 0;
            __syncthreads();
            // with fewer beams than groups, neighbouring groups are one: G = the power of two at or above W
            float thr = INFINITY;
            const int groups = NT / per;
            int fold = 1;
            while (groups / (2 * fold) >= W) fold *= 2;
            for (int i = 0; i < groups; i += fold) {
                float z = gmax[i];
                for (int f = 1; f < fold; ++f) z = fmaxf(z, gmax[i + f]);
                thr = fminf(thr, z);
            }
            const key_t worst = run[cur][W - 1];
            if (worst) thr = fmaxf(thr, key_value(worst));
            if (top >= thr && top > -INFINITY) {
#pragma unroll
                for (int q = 0; q < VPT; ++q)
#pragma unroll
                    for (int j = 0; j < EV; ++j)
                        if (v[q][j] >= thr && v[q][j] > -INFINITY) {
                            const int at = atomicAdd(&count, 1);
                            if (at < LIST)
                                list[at] = lin::argmax_key(v[q][j], static_cast<unsigned>(base + (q * NT + tid) * EV + j));
                        }
            }
            __syncthreads();
            const int n = count;
            if (tid < W) run[cur ^ 1][tid] = 0;
            __syncthreads();
            if (n <= LIST) {
                for (int i = tid; i < n + W; i += NT) {
                    const key_t k = i < n ? list[i] : run[cur][i - n];
                    if (!k) continue;
                    int rank = above(run[cur], W, k);
                    for (int j = 0; j < n && rank < W; ++j) rank += list[j] > k;
                    if (rank < W) run[cur ^ 1][rank] = k;
                }
                __syncthreads();
            } else {
                key_t prev = ~0ull;
                for (int s = 0; s < W; ++s) {
                    key_t best = 0;
#pragma unroll
                    for (int q = 0; q < VPT; ++q)
#pragma unroll
                        for (int j = 0; j < EV; ++j)
                            if (v[q][j] > -INFINITY) {
                                const key_t k = lin::argmax_key(v[q][j], static_cast<unsigned>(base + (q * NT + tid) * EV + j));
                                if (k < prev && k > best) best = k;
                            }
                    if (tid < W && run[cur][tid] < prev && run[cur][tid] > best) best = run[cur][tid];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
                    if (lane == 0) red_k[warp] = best;
                    __syncthreads();
                    best = red_k[0];
#pragma unroll
                    for (int i = 1; i < NWARP; ++i) best = max(best, red_k[i]);
                    if (tid == 0) run[cur ^ 1][s] = best;
                    prev = best;
                    __syncthreads();
                }
            }
            cur ^= 1;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, o);
            merge_ml(m, l, m2, l2);
        }
        if (lane == 0) {
            red_m[warp] = m;
            red_l[warp] = l;
        }
        if (__any_sync(0xFFFFFFFFu, bad) && lane == 0) atomicOr(p.status, ST_BEAM_LOGIT);
        __syncthreads();
        const long long at = row * p.chunks + ch;
        if (tid == 0) {
            for (int i = 1; i < NWARP; ++i) merge_ml(m, l, red_m[i], red_l[i]);
            p.ml[at] = make_float2(m, l);
        }
        if (tid < W) p.keys[at * W + tid] = run[cur][tid];
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
    for (int i = tid; i < W * W; i += NT) final_keys[i] = 0;
    __syncthreads();
    // a warp per beam: lse, the beam's W best logits, their totals
    for (int b = warp; b < W; b += NWARP) {
        const float sc = s_score[b];
        if (!(sc > -INFINITY)) continue;
        if (s_done[b]) {
            if (lane == 0) {
                final_keys[b * W] = lin::argmax_key(sc, static_cast<unsigned>(b * W));
                final_token[b * W] = max(p.eos, 0);
            }
            continue;
        }
        const long long at = static_cast<long long>(first_row + b) * p.chunks;
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < p.chunks; i += 32) {
            const float2 z = __ldcg(&p.ml[at + i]);
            merge_ml(m, l, z.x, z.y);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, o);
            // the same operands in the same order on both sides, so all lanes end alike
            if (lane & o) {
                float mm = m2, ll = l2;
                merge_ml(mm, ll, m, l);
                m = mm;
                l = ll;
            } else {
                merge_ml(m, l, m2, l2);
            }
        }
        const int n = p.chunks * W;
        for (int i = lane; i < n; i += 32) rowbuf[warp][i] = __ldcg(&p.keys[at * W + i]);
        __syncwarp();
        const float lse = m + logf(l);
        for (int i = lane; i < n; i += 32) {
            const key_t k = rowbuf[warp][i];
            if (!k) continue;
            int rank = 0;
            for (int c = 0; c < p.chunks && rank < W; ++c) rank += above(&rowbuf[warp][c * W], W, k);
            if (rank < W) {
                final_keys[b * W + rank] = lin::argmax_key(sc + (key_value(k) - lse), static_cast<unsigned>(b * W + rank));
                final_token[b * W + rank] = lin::argmax_key_index(k);
            }
        }
        __syncwarp();
    }
    __syncthreads();
    // the totals of a beam fall (rounding keeps the order; equal ones by rank), so these are sorted lists again
    for (int i = tid; i < W * W; i += NT) {
        const key_t k = final_keys[i];
        if (!k) continue;
        int rank = 0;
        for (int b = 0; b < W && rank < W; ++b) rank += above(&final_keys[b * W], W, k);
        if (rank < W) {
            const int out = first_row + rank, b = i / W;
            p.token[out] = final_token[i];
            p.parent[out] = first_row + b;
            p.new_score[out] = key_value(k);
            if (p.new_done) p.new_done[out] = s_done[b] || final_token[i] == p.eos;
        }
    }
    // fewer candidates than beams: the rest are dead
    int mine = 0;
    for (int i = tid; i < W * W; i += NT) mine += final_keys[i] != 0;
    int total = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
    if (lane == 0) red_l[warp] = static_cast<float>(mine);
    __syncthreads();
    for (int i = 0; i < NWARP; ++i) total += static_cast<int>(red_l[i]);
    if (tid >= total && tid < W) {
        const int out = first_row + tid;
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
static int launch(Params p, int B, int num_sms, cudaStream_t stream) {
    constexpr int EV = 16 / sizeof(T);
    const long long rows = static_cast<long long>(B) * p.W;
    // Tile: 4 vectors per thread where that still gives two CTAs per SM, else fewer, down to one: few rows are bound by
    // the latency of one CTA's work, many by bandwidth, which wants more loads in flight per thread.
    auto ctas = [&](int vpt) { return rows * ((p.V + NT * EV * vpt - 1) / (NT * EV * vpt)); };
    const int vpt = ctas(4) >= 2ll * num_sms ? 4 : ctas(2) >= 2ll * num_sms ? 2 : 1;
    const int tile = NT * EV * vpt, most = max_chunks(p.W);
    long long tiles = (p.V + tile - 1) / tile;
    const long long per = (tiles + most - 1) / most;  // tiles per chunk
    p.chunk = static_cast<int>(per * tile);
    p.chunks = static_cast<int>((tiles + per - 1) / per);
    const long long grid = rows * p.chunks;
    if (grid > 0x7FFFFFFFll) return GPT2_B200_EINVAL;
    auto *kern = vpt == 4 ? k_beam_select<T, 4> : vpt == 2 ? k_beam_select<T, 2> : k_beam_select<T, 1>;
    kern<<<static_cast<unsigned>(grid), NT, 0, stream>>>(p);
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
    return type == GPT2_BEAM_HALF ? beam::launch<__half>(p, B, ctx->num_sms, stream)
                                  : beam::launch<float>(p, B, ctx->num_sms, stream);
}
