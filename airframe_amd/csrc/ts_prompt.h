// ts_prompt.h -- launcher of the packed prompt attention (ts_prompt.hip).
#pragma once
#include "ts_packed.h"

namespace ts {

struct PromptCall {
    int32_t dtype;
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, k_stride, v_stride, out_stride;  // elements from one token's row to the next
    const int32_t *off;                                // host, [n_seq + 1]
    int n_seq, n_head, n_kv, hd;
    float softcap;
    void *ws;  // prompt_workspace bytes
};

// Scratch of a call over n_rows rows (f32: K and V split into two f16 planes; 0 otherwise).
uint64_t prompt_workspace(int32_t dtype, int64_t n_rows, int n_kv, int hd);
hipError_t launch_prompt(const PromptCall &c, hipStream_t st);

}  // namespace ts
