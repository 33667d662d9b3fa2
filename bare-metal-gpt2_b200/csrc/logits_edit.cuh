// logits_edit.cuh — the edit of logits and the greedy choice, as the decoder calls it (internal interface).
#pragma once
#include "common.cuh"

namespace b200 {
namespace edit {

// GPT2_B200_OK if an edit of rows of V logits may be launched.
int check(const GPT2LogitsEdit *e, int rows, int V);
// Kernel attributes on the current device (before a capture).
int prepare(DeviceContext *ctx);
// gpt2_logits_edit_b200 with len_add added to every length. With len_add and next, a row whose length is below its prompt's is left as it
// is, next too. pdl: a programmatic dependent of the kernel before it.
int launch(DeviceContext *ctx, void *out, long long ldo, const void *in, long long ld, int type, int rows, int V, const GPT2LogitsEdit &e, int len_add, int *next,
           bool pdl, cudaStream_t stream);

}  // namespace edit
}  // namespace b200
