// ts_shared.h -- launcher of attention behind a shared prefix (ts_shared.hip).
#pragma once
#include "ts_internal.h"

namespace ts {

// How a call divides its work: the prefix in n_part pieces of `chunk` keys (a multiple of 64) for
// every block of 128 (token, head) columns.
struct SharedPlan {
    int n_blk, n_part, chunk;
};
SharedPlan shared_plan(int n_rows, int G, int n_kv, int prefix_len, int stored_hd, int n_cu);
// The most pieces of any prefix up to max_prefix.
int shared_parts_cap(int n_rows, int G, int n_kv, int max_prefix, int stored_hd, int n_cu);

struct SharedCall {
    KvLayerView own, pre;
    int prefix_seq, prefix_len;
    const int32_t *d_len;
    const float *q;
    int n_head, n_tok;
    const float *rope;
    int rope_pairs, rope_rows;
    float softcap;
    float *out;
    SharedPlan plan;
    float *part;  // [n_seq n_tok n_head][n_part (+ 1: own keys, n_tok > 1)] of stored_hd + 2 floats
    // One token: the partials that the decode kernel wrote of the own keys, its plan, and the length
    // it was given with the launch (or -1).
    const float *own_part;
    DecodePlan own_plan;
    int hlen;
};
hipError_t launch_shared(const SharedCall &c, hipStream_t st);

}  // namespace ts
