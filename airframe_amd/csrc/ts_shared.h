// ts_shared.h -- launcher of attention behind a shared prefix (ts_shared.hip).
#pragma once
#include "ts_internal.h"

namespace ts {

// How a call divides its work.  chain: every block of 128 (token, head) columns of a sequence walks the
// prefix and then the sequence's own keys, and writes its output.  Otherwise the prefix in n_part pieces
// of `chunk` keys (a multiple of 64) for every block of columns of the whole batch, and (n_tok > 1)
// own_blk blocks of each sequence over its own keys, as partials that a last kernel joins.
struct SharedPlan {
    bool chain;
    int n_blk, n_part, chunk, own_blk;
};
SharedPlan shared_plan(int n_seq, int n_tok, int G, int n_kv, int prefix_len, int stored_hd, int n_cu);
// The most partials a row has, of any prefix up to max_prefix (0 for chains).
int shared_slots_cap(int n_seq, int n_tok, int G, int n_kv, int max_prefix, int n_cu);

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
    float *part;  // [n_seq n_tok n_head][n_part (+ 1 with own_blk)] of stored_hd + 2 floats
    // One token: where the decode kernel's partials of the own keys are, its plan, and the length it is
    // given with the launch (or -1).  own_here: its workgroups (the 16x16 kernel's, four waves or eight) go
    // out with the prefix's, with the new token's K and V to append, or null; otherwise they ran before.
    const float *own_part;
    DecodePlan own_plan;
    int hlen;
    bool own_here;
    const float *k_new, *v_new;
    int n_cu;
};
hipError_t launch_shared(const SharedCall &c, hipStream_t st);

}  // namespace ts
