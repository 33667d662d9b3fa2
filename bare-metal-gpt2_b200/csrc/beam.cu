// beam.cu — beam search with GPT-2-124M over the paged 8-bit cache.
//
// B prompts with W beams each are B x W rows of one cache. A step is the decode step of model.cu with
// the 8-bit cache in the place of the fp16 arenas, and the selection in the place of the argmax:
//   embedding + LayerNorm; per layer QKV linear, store of the step's K/V, attention, projection, LayerNorm, FC,
//   projection, LayerNorm; head with logits; selection; bookkeeping; reorder of the pages
// While a prompt lasts its item decodes in row b*W alone (the other rows are kept empty); its last token's
// selection forks that row's pages into W beams, which hold the whole pages of the prompt in common from then on. The
// step is captured in one CUDA graph and replayed, up to the last one, which is launched by itself: it makes no room behind it. Tokens and parents of every step are kept, and the
// hypotheses are read back from their ends.
#include <algorithm>
#include <new>

#include "model.cuh"

using namespace b200;
using namespace b200::model;

struct gpt2_b200_beam {
    int B = 0, W = 0, rows = 0, cap = 0, device = 0;
    GPT2WeightsGPU w;
    GPT2KV8Cache kv;
    void *arena = nullptr;
    __half *x = nullptr, *ln = nullptr, *qkv = nullptr, *att = nullptr, *fc = nullptr, *logits = nullptr;
    unsigned long long *amax = nullptr;
    int *tok = nullptr, *parent = nullptr, *done = nullptr, *sel_tok = nullptr, *sel_parent = nullptr, *sel_done = nullptr;
    float *score = nullptr, *sel_score = nullptr;
    int *step = nullptr;
    int2 *hist = nullptr;  // [cap + 1][rows]: token, beam it continues
    void *select_work = nullptr;
    size_t select_bytes = 0;
    lin::Plan qkv_p[NL], proj_p[NL], fc_p[NL], proj2_p[NL], head_p;
    cudaGraphExec_t graph = nullptr;
    const int *g_prompt = nullptr, *g_plen = nullptr;
    long long g_ps = 0;
    int g_eos = 0;
};

namespace {

constexpr int LDL = (V + 7) / 8 * 8;  // row stride of the logits

__global__ void k_beam_init(int *tok, float *score, int *done, int *step, const int *prompt, long long prompt_stride, int rows, int W) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r == 0) *step = 0;
    if (r >= rows) return;
    tok[r] = prompt[r / W * prompt_stride];
    score[r] = r % W ? -INFINITY : 0.0f;
    done[r] = 0;
}

// What the next step starts from: the prompt's next token while there is one, else the selection. One CTA.
__global__ void __launch_bounds__(256)
    k_beam_advance(int *tok, int *parent, float *score, int *done, const int *sel_tok, const int *sel_parent, const float *sel_score,
                   const int *sel_done, int2 *hist, int *step, const int *prompt, long long prompt_stride, const int *plen, int rows, int W) {
    const int r = threadIdx.x, next = *step + 1;
    __syncthreads();
    if (r == 0) *step = next;
    if (r >= rows) return;
    const int b = r / W, w = r - b * W;
    int t = sel_tok[r], from = sel_parent[r], d = sel_done[r];
    float s = sel_score[r];
    if (next < plen[b]) {
        t = prompt[b * prompt_stride + min(static_cast<long long>(next), prompt_stride - 1)];
        from = w ? -1 : r;
        s = w ? -INFINITY : 0.0f;
        d = 0;
    }
    tok[r] = t;
    parent[r] = from;
    score[r] = s;
    done[r] = d;
    hist[static_cast<long long>(next) * rows + r] = make_int2(t, from < 0 ? 0 : from - b * W);
}

// Hypothesis r from its end: one thread per row.
__global__ void k_beam_trace(int *out, long long out_stride, float *out_score, const float *score, const int2 *hist, const int *prompt,
                             long long prompt_stride, int n_steps, int rows, int W) {
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    const int b = r / W;
    int w = r - b * W;
    for (int t = n_steps; t >= 1; --t) {
        const int2 e = hist[static_cast<long long>(t) * rows + b * W + w];
        out[r * out_stride + t] = e.x;
        w = min(max(e.y, 0), W - 1);
    }
    out[r * out_stride] = prompt[b * prompt_stride];
    if (out_score) out_score[r] = score[r];
}

// One step; reserve: the positions to make room for behind it.
int enqueue(gpt2_b200_beam *bm, const int *prompt, long long ps, const int *plen, int eos, int reserve, cudaStream_t st) {
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_ECUDA;
    const GPT2WeightsGPU &w = bm->w;
    const GPT2KV8Cache *kv = &bm->kv;
    const int rows = bm->rows;
    int rc = launch(k_embed_ln, rows, LN_THREADS, st, false, bm->x, bm->ln, w.wte, w.wpe, w.layers[0].ln1_g, w.layers[0].ln1_b,
                    bm->tok, kv->len, bm->cap, ctx->status);
    for (int L = 0; L < NL && rc == GPT2_B200_OK; ++L) {
        const __half *g = L + 1 < NL ? w.layers[L + 1].ln1_g : w.lnf_g;
        const __half *bb = L + 1 < NL ? w.layers[L + 1].ln1_b : w.lnf_b;
        if ((rc = lin::launch_linear(bm->qkv_p[L], st)) || (rc = gpt2_kv8_store_b200(kv, L, 1, bm->qkv + E, bm->qkv + 2 * E, 0, Q, 0, nullptr, 1, st)) ||
            (rc = gpt2_kv8_attend_b200(bm->att, E, 0, bm->qkv, Q, 0, kv, L, NH, 1, nullptr, nullptr, 1, bm->cap, st)) ||
            (rc = lin::launch_linear(bm->proj_p[L], st)) ||
            (rc = launch(k_layernorm, rows, LN_THREADS, st, true, bm->ln, bm->x, w.layers[L].ln2_g, w.layers[L].ln2_b)) ||
            (rc = lin::launch_linear(bm->fc_p[L], st)) || (rc = lin::launch_linear(bm->proj2_p[L], st)) ||
            (rc = launch(k_layernorm, rows, LN_THREADS, st, true, bm->ln, bm->x, g, bb)))
            return rc;
    }
    if (rc || (rc = lin::launch_linear(bm->head_p, st)) ||
        (rc = gpt2_beam_select_b200(bm->sel_tok, bm->sel_parent, bm->sel_score, bm->sel_done, bm->logits, GPT2_BEAM_HALF, LDL, bm->score,
                                    bm->done, bm->B, bm->W, V, eos, bm->select_work, bm->select_bytes, st)) ||
        (rc = launch(k_beam_advance, 1, 256, st, false, bm->tok, bm->parent, bm->score, bm->done, bm->sel_tok, bm->sel_parent, bm->sel_score,
                     bm->sel_done, bm->hist, bm->step, prompt, ps, plen, rows, bm->W)))
        return rc;
    return gpt2_kv8_reorder_b200(kv, bm->parent, 1, reserve, st);
}

int beam_init(gpt2_b200_beam *bm, const GPT2WeightsGPU *w, const GPT2KV8Cache *kv, int B, int W) {
    if (!weights_ok(w) || !kv || B < 1 || W < 1 || W > 32 || B > lin::MAX_BPAD / W || kv->nRow != B * W || kv->nLayer != NL || kv->nHead != NH ||
        kv->headDim != HD || !kv->data || !kv->len || !gpt2_kv8_work_bytes_b200(kv, NH, 1) || kv->work_bytes < gpt2_kv8_work_bytes_b200(kv, NH, 1))
        return GPT2_B200_EINVAL;
    DeviceContext *ctx = device_context();
    if (!ctx) return GPT2_B200_EDEVICE;
    bm->B = B;
    bm->W = W;
    const int rows = bm->rows = B * W;
    bm->cap = static_cast<int>(std::min<long long>(static_cast<long long>(kv->maxPages) * kv->page, 1024));  // wpe has 1024 positions
    bm->device = ctx->device;
    bm->w = *w;
    bm->kv = *kv;
    const int head_tiles = (V + lin::BM - 1) / lin::BM;
    bm->select_bytes = gpt2_beam_work_bytes_b200(B, W);
    size_t total = 0;
    auto take = [&](size_t bytes) {
        const size_t at = total;
        total += (bytes + 255) & ~static_cast<size_t>(255);
        return at;
    };
    const size_t h = sizeof(__half) * rows, i4 = sizeof(int) * rows;
    const size_t o_x = take(h * E), o_ln = take(h * E), o_qkv = take(h * Q), o_att = take(h * E), o_fc = take(h * F), o_log = take(h * LDL);
    const size_t o_am = take(sizeof(unsigned long long) * rows * head_tiles), o_int = take(8 * ((i4 + 255) & ~static_cast<size_t>(255)));
    const size_t o_step = take(sizeof(int)), o_hist = take(sizeof(int2) * rows * (bm->cap + 1ull)), o_sel = take(bm->select_bytes);
    if (cudaMalloc(&bm->arena, total) != cudaSuccess) return GPT2_B200_ENOMEM;
    if (cudaMemset(bm->arena, 0, total) != cudaSuccess) return GPT2_B200_ECUDA;
    char *a = static_cast<char *>(bm->arena);
    bm->x = reinterpret_cast<__half *>(a + o_x);
    bm->ln = reinterpret_cast<__half *>(a + o_ln);
    bm->qkv = reinterpret_cast<__half *>(a + o_qkv);
    bm->att = reinterpret_cast<__half *>(a + o_att);
    bm->fc = reinterpret_cast<__half *>(a + o_fc);
    bm->logits = reinterpret_cast<__half *>(a + o_log);
    bm->amax = reinterpret_cast<unsigned long long *>(a + o_am);
    char *ints = a + o_int;
    auto next = [&] {
        int *p = reinterpret_cast<int *>(ints);
        ints += (i4 + 255) & ~static_cast<size_t>(255);
        return p;
    };
    bm->tok = next();
    bm->parent = next();
    bm->done = next();
    bm->sel_tok = next();
    bm->sel_parent = next();
    bm->sel_done = next();
    bm->score = reinterpret_cast<float *>(next());
    bm->sel_score = reinterpret_cast<float *>(next());
    bm->step = reinterpret_cast<int *>(a + o_step);
    bm->hist = reinterpret_cast<int2 *>(a + o_hist);
    bm->select_work = a + o_sel;
    int rc = GPT2_B200_OK;
    for (int L = 0; L < NL; ++L) {
        const GPT2LayerGPU &l = w->layers[L];
        if ((rc = lin::plan_linear(&bm->qkv_p[L], lin::EPI_STORE, l.qkv_w, Q, E, bm->ln, E, rows, l.qkv_b, bm->qkv, Q, 0, ctx->num_sms)) ||
            (rc = lin::plan_linear(&bm->proj_p[L], lin::EPI_RESID, l.attn_proj_w, E, E, bm->att, E, rows, l.attn_proj_b, bm->x, E, 0, ctx->num_sms)) ||
            (rc = lin::plan_linear(&bm->fc_p[L], lin::EPI_GELU, l.fc_w, F, E, bm->ln, E, rows, l.fc_b, bm->fc, F, 0, ctx->num_sms)) ||
            (rc = lin::plan_linear(&bm->proj2_p[L], lin::EPI_RESID, l.proj_w, E, F, bm->fc, F, rows, l.proj_b, bm->x, E, 0, ctx->num_sms)))
            return rc;
        for (lin::Plan *p : {&bm->qkv_p[L], &bm->proj_p[L], &bm->fc_p[L], &bm->proj2_p[L]}) {
            p->pdl = true;  // weight tiles are requested while the kernel before ends
            if ((rc = lin::prepare_linear(*p))) return rc;
        }
    }
    if ((rc = lin::plan_linear(&bm->head_p, lin::EPI_HEAD, w->wte, V, E, bm->ln, E, rows, nullptr, bm->logits, LDL, 1, ctx->num_sms)))
        return rc;
    bm->head_p.p.amax = bm->amax;
    bm->head_p.pdl = true;
    return lin::prepare_linear(bm->head_p);
}

}  // namespace

extern "C" {

int gpt2_b200_beam_create(gpt2_b200_beam **out, const GPT2WeightsGPU *w, const GPT2KV8Cache *kv, int B, int W) {
    if (!out) return GPT2_B200_EINVAL;
    *out = nullptr;
    gpt2_b200_beam *bm = new (std::nothrow) gpt2_b200_beam();
    if (!bm) return GPT2_B200_ENOMEM;
    const int rc = beam_init(bm, w, kv, B, W);
    if (rc != GPT2_B200_OK) {
        gpt2_b200_beam_destroy(bm);
        return rc;
    }
    *out = bm;
    return GPT2_B200_OK;
}

void gpt2_b200_beam_destroy(gpt2_b200_beam *bm) {
    if (!bm) return;
    if (bm->arena) {  // replays queued on any stream may still be running
        int prev = -1;
        if (cudaGetDevice(&prev) == cudaSuccess && prev != bm->device) cudaSetDevice(bm->device);
        cudaDeviceSynchronize();
        if (bm->graph) cudaGraphExecDestroy(bm->graph);
        cudaFree(bm->arena);
        if (prev >= 0 && prev != bm->device) cudaSetDevice(prev);
    }
    delete bm;
}

int gpt2_b200_beam_generate(gpt2_b200_beam *bm, const int *d_prompt, long long prompt_stride, const int *d_plen, int n_steps, int eos,
                            int *d_out, long long out_stride, float *d_score, cudaStream_t stream) {
    if (!bm || !d_prompt || !d_plen || !d_out || n_steps < 1 || n_steps > bm->cap || out_stride < n_steps + 1 || prompt_stride < 1 ||
        eos < -1 || eos >= V)
        return GPT2_B200_EINVAL;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) return GPT2_B200_ECUDA;
    if (dev != bm->device) return GPT2_B200_EINVAL;
    if (bm->graph && (bm->g_prompt != d_prompt || bm->g_plen != d_plen || bm->g_ps != prompt_stride || bm->g_eos != eos)) {
        // earlier replays may still be queued: let them finish first
        if (cudaDeviceSynchronize() != cudaSuccess) return GPT2_B200_ECUDA;
        cudaGraphExecDestroy(bm->graph);
        bm->graph = nullptr;
    }
    bm->g_prompt = d_prompt;
    bm->g_plen = d_plen;
    bm->g_ps = prompt_stride;
    bm->g_eos = eos;
    int rc = GPT2_B200_OK;
    if (!bm->graph) {
        cudaStream_t cs;
        if (cudaStreamCreateWithFlags(&cs, cudaStreamNonBlocking) != cudaSuccess) return GPT2_B200_ECUDA;
        cudaGraph_t g = nullptr;
        if (cudaStreamBeginCapture(cs, cudaStreamCaptureModeThreadLocal) != cudaSuccess) {
            rc = GPT2_B200_ECUDA;
        } else {
            rc = enqueue(bm, d_prompt, prompt_stride, d_plen, eos, 1, cs);
            if (cudaStreamEndCapture(cs, &g) != cudaSuccess && rc == GPT2_B200_OK) rc = GPT2_B200_ECUDA;
        }
        if (rc == GPT2_B200_OK && cudaGraphInstantiate(&bm->graph, g, 0) != cudaSuccess) rc = GPT2_B200_ECUDA;
        if (g) cudaGraphDestroy(g);
        cudaStreamDestroy(cs);
        if (rc != GPT2_B200_OK) {
            bm->graph = nullptr;
            return rc;
        }
    }
    const int blocks = (bm->rows + 127) / 128;
    if ((rc = gpt2_kv8_reset_b200(&bm->kv, stream)) || (rc = gpt2_kv8_reorder_b200(&bm->kv, nullptr, 0, 1, stream))) return rc;
    k_beam_init<<<blocks, 128, 0, stream>>>(bm->tok, bm->score, bm->done, bm->step, d_prompt, prompt_stride, bm->rows, bm->W);
    if (cudaGetLastError() != cudaSuccess) return GPT2_B200_ECUDA;
    for (int s = 1; s < n_steps; ++s)
        if (cudaGraphLaunch(bm->graph, stream) != cudaSuccess) return GPT2_B200_ECUDA;
    // The last step leaves no room behind it, for which table and pool need not have pages.
    if ((rc = enqueue(bm, d_prompt, prompt_stride, d_plen, eos, 0, stream))) return rc;
    k_beam_trace<<<blocks, 128, 0, stream>>>(d_out, out_stride, d_score, bm->score, bm->hist, d_prompt, prompt_stride, n_steps, bm->rows,
                                            bm->W);
    return cudaGetLastError() == cudaSuccess ? GPT2_B200_OK : GPT2_B200_ECUDA;
}

}  // extern "C"
