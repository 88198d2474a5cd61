// ts_evict_ops.cpp -- host side of cache eviction: argument checks and dispatch.
#include "ts_evict.h"

#include <math.h>

#include <cmath>
#include <memory>
#include <new>

#include "ts_host.h"

using namespace ts;

// Whether two ranges of bytes share memory (an empty one never does).
static bool shares(const void *a, uint64_t na, const void *b, uint64_t nb) {
    return a && b && na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

static bool aligned4(const void *p) { return ((uintptr_t)p & 3u) == 0; }

// Rows of weights of one layer, in bytes.
static uint64_t weight_bytes(const ts_kv *kv) { return (uint64_t)kv->d.n_seq * kv->d.n_head_kv * kv->d.max_seq * sizeof(float); }

extern "C" {

// (work-items of a launch are a 32-bit number, sequences its second dimension)
static bool weigh_shape_ok(const ts_kv *kv, int32_t n_head, int32_t n_tok) {
    return kv && heads_ok(kv, n_head) && n_head / kv->d.n_head_kv <= 4096 && n_tok >= 0 && kv->d.n_seq <= 65535 &&
           (int64_t)kv->d.n_seq * n_tok * n_head <= (n_tok == 1 ? UINT32_MAX / 256 : UINT32_MAX / 128);
}

int ts_attn_weigh_workspace(const ts_kv *kv, int32_t n_head, int32_t n_tok, uint64_t *bytes) {
    if (!bytes || !weigh_shape_ok(kv, n_head, n_tok)) return TS_ERR_INVALID;
    *bytes = 0;
    if (n_tok == 0) return TS_OK;
    if (n_tok > 1) {
        *bytes = weigh_chunk_workspace(kv->d.n_seq, n_tok, n_head, kv->d.n_head_kv, kv->hdp, kv->d.max_seq, kv->n_cu);
        return TS_OK;
    }
    *bytes = weigh_token_workspace(kv->d.n_seq, n_head, kv->d.n_head_kv, kv->P, kv->d.max_seq, kv->hdp, kv->n_cu);
    return TS_OK;
}

int ts_attn_weigh(ts_kv *kv, int32_t layer, const float *d_k, const float *d_v, const float *d_q, int32_t n_head,
                  int32_t n_tok, const ts_rope *rope, float softcap, float *d_weights, int32_t fresh, float *d_out,
                  void *d_workspace, uint64_t workspace_bytes, void *stream) {
    if (!weigh_shape_ok(kv, n_head, n_tok) || layer < 0 || layer >= kv->d.n_layers || !(softcap >= 0.0f) ||
        !std::isfinite(softcap) || (d_k == nullptr) != (d_v == nullptr) || (d_k && n_tok != 1) || !aligned16(d_k) ||
        !aligned16(d_v) || (fresh != 0 && fresh != 1))
        return TS_ERR_INVALID;
    if (n_tok == 0) return TS_OK;
    if (!d_q || !d_out || !d_weights || !aligned16(d_q) || !aligned16(d_out) || !aligned4(d_weights)) return TS_ERR_INVALID;
    const int32_t max_len = *std::max_element(kv->h_len.begin(), kv->h_len.end());
    if ((int64_t)max_len + n_tok > kv->d.max_seq) return TS_ERR_OVERFLOW;
    const int rc = check_rope(rope, kv->d.head_dim, rot_end(kv, n_tok));
    if (rc) return rc;
    uint64_t need = 0;
    ts_attn_weigh_workspace(kv, n_head, n_tok, &need);
    if (!d_workspace || workspace_bytes < need) return TS_ERR_WORKSPACE;
    if (!aligned16(d_workspace)) return TS_ERR_INVALID;
    // every launch of the call reads its inputs: what it writes is apart from them and from each other
    const uint64_t qb = (uint64_t)kv->d.n_seq * n_tok * n_head * kv->d.head_dim * sizeof(float);
    const uint64_t kb = qb / n_head * kv->d.n_head_kv, wb = weight_bytes(kv);
    const struct { const void *p; uint64_t n; } arg[6] = {{d_out, qb}, {d_weights, wb}, {d_workspace, need}, {d_q, qb}, {d_k, kb}, {d_v, kb}};
    for (int i = 0; i < 3; i++)
        for (int j = i + 1; j < 6; j++)
            if (shares(arg[i].p, arg[i].n, arg[j].p, arg[j].n)) return TS_ERR_INVALID;

    WeighCall c;
    c.L = rotating_layer(kv, layer, rope, stream);
    c.d_len = kv->d_len;
    for (int s = 0; s < kv->d.n_seq; s++) kv->h_ctx[s] = kv->h_len[s] + n_tok;
    c.n_ctx = kv->h_ctx.data();
    c.own_max = max_len + n_tok;
    c.captured = capturing(stream) || kv->len_captured;
    c.q = d_q;
    c.n_head = n_head;
    c.n_tok = n_tok;
    c.rope = rope->d_table;
    c.rope_pairs = rope->rope_dim / 2;
    c.rope_rows = rope->n_pos;
    c.softcap = softcap;
    c.out = d_out;
    c.max_seq = kv->d.max_seq;
    c.w = d_weights;
    c.fresh = fresh != 0;
    c.n_cu = kv->n_cu;
    c.ws = static_cast<uint8_t *>(d_workspace);
    if (n_tok > 1) return hip_status(launch_weigh_chunk(c, as_stream(stream)));
    c.k_new = d_k;
    c.v_new = d_v;
    // (an eager call gives a lone sequence's length with the launch, as ts_attn_decode)
    c.hlen = kv->d.n_seq == 1 && !c.captured ? kv->h_len[0] : -1;
    DecodePlan plan = decode_plan(kv->h_ctx.data(), kv->d.n_seq, kv->d.n_head_kv, n_head / kv->d.n_head_kv, kv->n_cu,
                                  kv->hdp, d_k != nullptr);
    // The integer kernel runs a workgroup per CU, those past a short sequence's end too, and the grid is a rectangle of
    // sequences by the longest one's splits: of a ragged batch, longer splits whose rectangle fits the CUs in one round, if no longer
    // than 5/2 of the plan's.  4 sequences of 700-6001 slots of 256-dim heads 28.5 us, 19.6 so; 8 of 1001-16003 with 128
    // dims 30.7 and 26.2, with 8 query heads per kv head 42.6 and 34.7.  (Of the first two's 256 workgroups 120 have keys.)
    const int round = kv->n_cu / (kv->d.n_seq * kv->d.n_head_kv);
    if (plan.g4 && round > 1 && plan.n_split > round) {
        const int chunk = ((c.own_max + round - 1) / round + 63) / 64 * 64;
        if (2 * (int64_t)chunk <= 5 * (int64_t)plan.chunk) {
            plan.chunk = chunk;
            plan.n_split = (c.own_max + chunk - 1) / chunk;
        }
    }
    return hip_status(launch_weigh_token(c, plan, as_stream(stream)));
}

int ts_kv_select(const ts_kv *kv, const float *d_weights, int32_t keep, int32_t n_sink, int32_t n_recent, int32_t *d_slots,
                 void *stream) {
    if (!kv || keep <= 0 || keep > kv->d.max_seq || n_sink < 0 || n_recent < 0 || (int64_t)n_sink + n_recent > keep ||
        !d_weights || !d_slots || !aligned4(d_weights) || !aligned4(d_slots))
        return TS_ERR_INVALID;
    const uint64_t rows = (uint64_t)kv->d.n_layers * kv->d.n_seq * kv->d.n_head_kv;
    // (a row's bytes and a layer's work-items are 32-bit numbers)
    if (rows / kv->d.n_layers > UINT32_MAX / 1024 || kv->d.max_seq > (1 << 28)) return TS_ERR_INVALID;
    if (shares(d_weights, weight_bytes(kv) * kv->d.n_layers, d_slots, rows * keep * sizeof(int32_t))) return TS_ERR_INVALID;
    const int max_len = *std::max_element(kv->h_len.begin(), kv->h_len.end());
    return hip_status(launch_select(d_weights, kv->d_len, max_len, kv->d.n_layers, kv->d.n_seq, kv->d.n_head_kv, kv->d.max_seq, keep,
                                    n_sink, n_recent, d_slots, as_stream(stream)));
}

int ts_kv_keep(ts_kv *dst, int32_t dst_seq, const ts_kv *src, int32_t src_seq, int32_t n_seq, const int32_t *d_slots,
               int32_t keep, const float *d_src_weights, float *d_weights, void *stream) {
    if (!dst || !src || n_seq < 0 || dst_seq < 0 || src_seq < 0 || (int64_t)dst_seq + n_seq > dst->d.n_seq ||
        (int64_t)src_seq + n_seq > src->d.n_seq || dst->d.n_layers != src->d.n_layers || dst->d.n_head_kv != src->d.n_head_kv ||
        dst->d.head_dim != src->d.head_dim || dst->device != src->device || keep <= 0 || !aligned4(d_slots) ||
        (d_src_weights == nullptr) != (d_weights == nullptr) || !aligned4(d_src_weights) || !aligned4(d_weights))
        return TS_ERR_INVALID;
    if (n_seq == 0) return TS_OK;
    if (!d_slots) return TS_ERR_INVALID;
    // in place, or into sequences apart from those that are read
    const bool in_place = dst == src && dst_seq == src_seq;
    if (dst == src && !in_place && dst_seq < src_seq + n_seq && src_seq < dst_seq + n_seq) return TS_ERR_INVALID;
    const uint64_t rows = (uint64_t)src->d.n_layers * n_seq * src->d.n_head_kv, slot_bytes = rows * keep * sizeof(int32_t);
    // (a layer's work-items are a 32-bit number: 64 of each of up to 9 slices of a row, elsewhere of its windows of 64 slots)
    const uint64_t windows = in_place ? 1 : ((uint64_t)std::min(keep, dst->d.max_seq) + 63) / 64;
    if (rows / src->d.n_layers * windows > UINT32_MAX / (9 * 64)) return TS_ERR_INVALID;
    const uint64_t sb = weight_bytes(src) * src->d.n_layers, db = weight_bytes(dst) * dst->d.n_layers;
    if (!(dst == src && d_weights == d_src_weights) && shares(d_src_weights, sb, d_weights, db)) return TS_ERR_INVALID;
    if (shares(d_slots, slot_bytes, d_weights, db)) return TS_ERR_INVALID;
    if (capturing(stream)) return TS_ERR_INVALID;  // (the host's lengths change with the call)
    // Lengths, bases and sinks as the device has them: replays of a captured call move them past the host's.
    const int32_t *h_len = src->h_len.data(), *h_rot = src->h_rot.data(), *h_sink = src->h_sink.data();
    std::unique_ptr<int32_t[]> now;
    if (src->len_captured) {
        const size_t ints = 3 * (size_t)src->d.n_seq;
        now.reset(new (std::nothrow) int32_t[ints]);
        if (!now) return TS_ERR_NOMEM;
        if (hipMemcpyAsync(now.get(), src->d_len, ints * sizeof(int32_t), hipMemcpyDeviceToHost, as_stream(stream)) != hipSuccess ||
            hipStreamSynchronize(as_stream(stream)) != hipSuccess)
            return TS_ERR_HIP;
        h_len = now.get();
        h_rot = h_len + src->d.n_seq;
        h_sink = h_rot + src->d.n_seq;
    }
    for (int i = 0; i < n_seq; i++) {
        const int s = src_seq + i, len = std::min(h_len[s], src->d.max_seq), n = std::min(len, keep);
        if (h_sink[s] != 0) return TS_ERR_INVALID;  // (sinks are rotated at their own slot, the others past the window base)
        if (n > dst->d.max_seq || (int64_t)h_rot[s] + len - n > INT32_MAX / 2) return TS_ERR_OVERFLOW;
    }
    KeepCall c;
    c.src = src->layer(0);
    c.dst = dst->layer(0);
    c.src_layer = src->layer_bytes;
    c.dst_layer = dst->layer_bytes;
    c.src_len = src->d_len;
    c.src_rot = src->d_rot;
    c.dst_len = dst->d_len;
    c.dst_rot = dst->d_rot;
    c.dst_sink = dst->d_sink;
    c.src_seq = src_seq;
    c.dst_seq = dst_seq;
    c.n_seq = n_seq;
    c.n_layers = src->d.n_layers;
    c.first_layer = 0;
    c.keep = std::min(keep, dst->d.max_seq);
    c.slot_row = keep;
    c.src_max = src->d.max_seq;
    c.dst_max = dst->d.max_seq;
    c.in_place = in_place;
    c.slots = d_slots;
    c.src_w = d_src_weights;
    c.dst_w = d_weights;
    if (launch_keep(c, as_stream(stream)) != hipSuccess) return TS_ERR_HIP;
    for (int i = 0; i < n_seq; i++) {
        const int s = src_seq + i, d = dst_seq + i, len = std::min(h_len[s], src->d.max_seq), n = std::min(len, keep);
        dst->h_rot[d] = h_rot[s] + len - n;
        dst->h_len[d] = n;
        dst->h_sink[d] = 0;
    }
    return TS_OK;
}

}  // extern "C"
