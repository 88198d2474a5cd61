// ts_shared.h -- launcher of attention behind a shared prefix (ts_shared.hip).
#pragma once
#include "ts_internal.h"

namespace ts {

// How a call divides its work.  chain: every block of 128 (token, head) columns of a sequence walks the
// prefix and then the sequence's own keys, and writes its output.  Otherwise the prefix in n_part pieces
// of `chunk` keys (a multiple of 64) for every block of columns of the whole batch, and (n_tok > 1)
// own_blk blocks of each sequence over its own keys, own_pieces pieces of own_chunk keys, as partials that a
// last kernel joins.
struct SharedPlan {
    bool chain;
    int n_blk, n_part, chunk, own_blk, own_pieces, own_chunk;
};
// own_max: the longest sequence's own keys, the new tokens' included.
SharedPlan shared_plan(int n_seq, int n_tok, int G, int n_kv, int prefix_len, int own_max, int n_cu);
// The splits of the own keys (n_ctx of them) for one token.
void shared_own_plan(const int32_t *n_ctx, int n_seq, int n_kv, int G, int n_cu, int *chunk, int *n_split);
// The most partials a row has, of any prefix up to max_prefix and own keys up to own_max (0 for chains).
int shared_slots_cap(int n_seq, int n_tok, int G, int n_kv, int max_prefix, int own_max, int n_cu);

// The plan of a chunk over its own keys alone (no prefix; weighed attention), n_ctx of them with the new tokens: as
// many pieces as fill the chip, a chain if that is one.  own_pieces_cap: the most pieces of any lengths up to own_max.
SharedPlan own_plan(const int32_t *n_ctx, int n_seq, int n_tok, int G, int n_kv, int n_cu);
int own_pieces_cap(int n_seq, int n_tok, int G, int n_kv, int own_max, int n_cu);

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
    float *part;  // [n_seq n_tok n_head][n_part (+ own_pieces with own_blk)] of stored_hd + 2 floats
    // One token: the own keys go out as splits of the 16x16 decode kernel beside the prefix's pieces, their
    // partials in own_part (null for a chunk), with the new token's K and V to append, or null; hlen: the
    // sequence's length where the launch gives it (or -1).
    float *own_part;
    int own_chunk, own_split;
    int hlen;
    const float *k_new, *v_new;
    int n_cu;
    // [n_seq][n_head_kv][n_blk32] ColBlock: the columns are left there too, a chain's with their log2 sums, and
    // the partials of pieces are the caller's to join (null: not wanted).
    void *cols = nullptr;
    int n_blk32 = 0;
};
hipError_t launch_shared(const SharedCall &c, hipStream_t st);

}  // namespace ts
