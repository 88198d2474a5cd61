// ts_evict.h -- launchers of cache eviction: attention that adds up what every slot receives
// (ts_weigh.hip), the choice of the slots that stay and their rows moved together (ts_evict.hip).
#pragma once
#include "ts_internal.h"

namespace ts {

struct WeighCall {
    KvLayerView L;
    const int32_t *d_len;
    const int32_t *n_ctx;  // slots of every sequence with the new tokens', as the host knows them, and the most of them
    int own_max;
    bool captured;  // (replays go past own_max)
    const float *q;
    int n_head, n_tok;
    const float *rope;
    int rope_pairs, rope_rows;
    float softcap;
    float *out;
    int max_seq;  // a row of weights
    float *w;     // [n_seq][n_head_kv][max_seq]
    bool fresh;
    int n_cu;
    uint8_t *ws;
    // one token: its K and V to append, or null; the sequence's length where the launch gives it (or -1)
    const float *k_new, *v_new;
    int hlen;
};
// One token.
uint64_t weigh_token_workspace(int n_seq, int n_head, int n_kv, int P, int max_seq, int stored_hd, int n_cu);
hipError_t launch_weigh_token(const WeighCall &c, const DecodePlan &plan, hipStream_t st);
// Chunks (n_tok > 1).
uint64_t weigh_chunk_workspace(int n_seq, int n_tok, int n_head, int n_kv, int stored_hd, int max_seq, int n_cu);
hipError_t launch_weigh_chunk(const WeighCall &c, hipStream_t st);

// Which slots stay: d_slots [n_layers][n_seq][H][keep] from w [n_layers][n_seq][H][max_seq].  max_len: the longest
// sequence as far as the host knows it (the choice of a kernel; any is right).
hipError_t launch_select(const float *w, const int32_t *d_len, int max_len, int n_layers, int n_seq, int H, int max_seq,
                         int keep, int n_sink, int n_recent, int32_t *d_slots, hipStream_t st);

struct KeepCall {
    KvLayerView src, dst;  // layer 0 of each
    uint64_t src_layer, dst_layer;  // bytes from layer to layer
    const int32_t *src_len, *src_rot;
    int32_t *dst_len, *dst_rot, *dst_sink;
    int src_seq, dst_seq, n_seq, n_layers, keep, src_max, dst_max;
    int first_layer;  // of a launch; slots and weights begin at it
    int slot_row;  // slots of a row of d_slots (keep, or more than fit the destination)
    bool in_place;
    const int32_t *slots;
    const float *src_w;
    float *dst_w;
};
// The rows, and then the lengths and window bases of the sequences they went to.
hipError_t launch_keep(const KeepCall &c, hipStream_t st);

}  // namespace ts
