// ts_ops.cpp -- host side of the packed-batch and shared-prefix entry points: argument checks and dispatch.
#include "ts_packed.h"

#include <math.h>

#include <cmath>
#include <new>

#include "ts_host.h"
#include "ts_prompt.h"
#include "ts_shared.h"

using namespace ts;

// Rows that 16-byte pieces reach: the first address and the distance from row to row.
static bool rows_ok(const void *p, int64_t stride, int64_t row, int32_t dtype) {
    return p && aligned16(p) && stride >= row && stride <= INT64_MAX / 16 / (int64_t)INT32_MAX &&
           stride * dtype_size(dtype) % 16 == 0;
}

// Whether rows first .. last - 1 of `row` bytes at two addresses, a_stride and b_stride bytes apart, share memory (rows
// that interleave at one stride do not; of different strides, where the ranges do).
static bool rows_overlap(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int64_t row, int64_t first,
                         int64_t last) {
    const int64_t a0 = (int64_t)(uintptr_t)a + first * a_stride, b0 = (int64_t)(uintptr_t)b + first * b_stride;
    const int64_t n = last - first - 1;
    if (a0 + n * a_stride + row <= b0 || b0 + n * b_stride + row <= a0) return false;
    if (a_stride != b_stride) return true;
    const int64_t d = (a0 > b0 ? a0 - b0 : b0 - a0) % a_stride;
    return d < row || d > a_stride - row;
}

// Whether two ranges of bytes share memory (one of no bytes, such as a workspace that is not needed: never).
static bool bytes_overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
    return a && b && na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// The largest length of a sequence after its rows of a packed batch, and its last rotation position.
static void packed_ends(const ts_kv *kv, const int32_t *off, int64_t &len_end, int64_t &rot_last) {
    len_end = rot_last = 0;
    for (int s = 0; s < kv->d.n_seq; s++) {
        const int64_t n = (int64_t)off[s + 1] - off[s];
        if (n == 0) continue;
        len_end = std::max(len_end, kv->h_len[s] + n);
        rot_last = std::max(rot_last, (int64_t)kv->h_len[s] + kv->h_rot[s] + n);
    }
}

extern "C" {

int ts_rope_create_scaled(int32_t n_pos, int32_t rope_dim, double base, double factor, int32_t l_train, double alpha,
                          double beta, double mult, ts_rope **out) {
    if (!out) return TS_ERR_INVALID;
    *out = nullptr;
    if (n_pos <= 0 || rope_dim <= 0 || (rope_dim & 1) || !(base > 0.0) || !std::isfinite(base) || !(factor > 0.0) ||
        !std::isfinite(factor) || !(mult > 0.0) || !std::isfinite(mult) || !(alpha >= 0.0) || !(beta >= 0.0) ||
        !std::isfinite(alpha) || !std::isfinite(beta) || (beta > alpha && l_train <= 0))
        return TS_ERR_INVALID;
    ts_rope *r = new (std::nothrow) ts_rope();
    if (!r) return TS_ERR_NOMEM;
    if (hipMalloc(&r->d_table, (size_t)n_pos * rope_dim * sizeof(float)) != hipSuccess) {
        delete r;
        return TS_ERR_NOMEM;
    }
    // (the table is whole when this returns, whatever stream reads it then)
    hipError_t e = launch_rope_table(r->d_table, n_pos, rope_dim, base, factor, l_train, alpha, beta, mult, nullptr);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
    if (e != hipSuccess) {
        (void)hipFree(r->d_table);
        delete r;
        return TS_ERR_HIP;
    }
    r->n_pos = n_pos;
    r->rope_dim = rope_dim;
    *out = r;
    return TS_OK;
}

int ts_rope_apply(const ts_rope *rope, int32_t layout, int32_t dtype, const void *d_x, int64_t x_stride,
                  const int32_t *d_pos, int32_t n_tok, int32_t n_head, int32_t head_dim, void *d_out, int64_t out_stride,
                  void *stream) {
    if (!rope || !dtype_ok(dtype) || (layout != TS_ROPE_INTERLEAVED && layout != TS_ROPE_HALF) || n_tok < 0 || n_head <= 0 ||
        head_dim <= 0 || head_dim % 8 != 0 || head_dim > 65536 || n_head > 65536 || rope->rope_dim > head_dim)
        return TS_ERR_INVALID;
    if (n_tok == 0) return TS_OK;
    const int64_t row = (int64_t)n_head * head_dim;
    if (row > (1 << 28)) return TS_ERR_INVALID;  // (a token's work items are 32-bit numbers)
    if (!d_pos || ((uintptr_t)d_pos & 3u) != 0 || !rows_ok(d_x, x_stride, row, dtype) || !rows_ok(d_out, out_stride, row, dtype))
        return TS_ERR_INVALID;
    // in place, or apart: a thread reads its rows before it writes them, but not before others write
    const int size = dtype_size(dtype);
    const uint8_t *x0 = (const uint8_t *)d_x, *o0 = (const uint8_t *)d_out;
    const uint8_t *x1 = x0 + ((n_tok - 1) * x_stride + row) * size, *o1 = o0 + ((n_tok - 1) * out_stride + row) * size;
    if (x0 == o0 ? x_stride != out_stride && n_tok > 1 : x0 < o1 && o0 < x1) return TS_ERR_INVALID;
    return hip_status(launch_rope_apply(dtype, layout, d_x, x_stride, d_pos, n_tok, n_head, head_dim, rope->d_table,
                                        rope->rope_dim / 2, rope->n_pos, d_out, out_stride, as_stream(stream)));
}

int ts_append_packed(ts_kv *kv, int32_t layer, int32_t dtype, const void *d_k, int64_t k_stride, const void *d_v,
                     int64_t v_stride, const int32_t *tok_off, const ts_rope *rope, void *stream) {
    if (!kv || layer < 0 || layer >= kv->d.n_layers || !dtype_ok(dtype) || !offsets_ok(tok_off, kv->d.n_seq))
        return TS_ERR_INVALID;
    if (tok_off[kv->d.n_seq] == tok_off[0]) return TS_OK;
    const int64_t row = (int64_t)kv->d.n_head_kv * kv->d.head_dim;
    if (!rows_ok(d_k, k_stride, row, dtype) || !rows_ok(d_v, v_stride, row, dtype)) return TS_ERR_INVALID;
    int64_t len_end, rot_last;
    packed_ends(kv, tok_off, len_end, rot_last);
    if (len_end > kv->d.max_seq) return TS_ERR_OVERFLOW;
    if (rope) {
        const int rc = check_rope(rope, kv->d.head_dim, rot_last);
        if (rc) return rc;
    }
    KvLayerView L = rotating_layer(kv, layer, rope, stream);
    if (!rope) L.qn = L.kn = nullptr;  // (K as it is stored: normalized and rotated by the caller)
    return hip_status(launch_append_packed(L, kv->d_len, dtype, d_k, k_stride, d_v, v_stride, tok_off,
                                           rope ? rope->d_table : nullptr, rope ? rope->rope_dim / 2 : 0,
                                           rope ? rope->n_pos : INT32_MAX, as_stream(stream)));
}

int ts_read_packed(const ts_kv *kv, int32_t layer, const int32_t *pos0, const int32_t *row_off, int32_t dtype, void *d_k,
                   int64_t k_stride, void *d_v, int64_t v_stride, void *stream) {
    if (!kv || layer < 0 || layer >= kv->d.n_layers || !dtype_ok(dtype) || !offsets_ok(row_off, kv->d.n_seq))
        return TS_ERR_INVALID;
    if (row_off[kv->d.n_seq] == row_off[0]) return TS_OK;
    const int64_t row = (int64_t)kv->d.n_head_kv * kv->d.head_dim;
    if (!rows_ok(d_k, k_stride, row, dtype) || !rows_ok(d_v, v_stride, row, dtype)) return TS_ERR_INVALID;
    const int size = dtype_size(dtype);
    if (rows_overlap(d_k, k_stride * size, d_v, v_stride * size, row * size, row_off[0], row_off[kv->d.n_seq]))
        return TS_ERR_INVALID;
    for (int s = 0; s < kv->d.n_seq; s++) {
        const int64_t p = pos0 ? pos0[s] : 0, n = (int64_t)row_off[s + 1] - row_off[s];
        if (n > 0 && (p < 0 || p + n > kv->d.max_seq)) return TS_ERR_INVALID;
    }
    return hip_status(launch_read_packed(kv->layer(layer), pos0, row_off, dtype, d_k, k_stride, d_v, v_stride,
                                         as_stream(stream)));
}

int ts_kv_increment_packed(ts_kv *kv, const int32_t *tok_off, void *stream) {
    if (!kv || !offsets_ok(tok_off, kv->d.n_seq)) return TS_ERR_INVALID;
    for (int s = 0; s < kv->d.n_seq; s++)
        if ((int64_t)kv->h_len[s] + tok_off[s + 1] - tok_off[s] > kv->d.max_seq) return TS_ERR_OVERFLOW;
    if (tok_off[kv->d.n_seq] == tok_off[0]) return TS_OK;
    note_len_change(kv, stream);
    const hipError_t e = launch_len_add(kv->d_len, kv->d.n_seq, tok_off, as_stream(stream));
    if (e != hipSuccess) return TS_ERR_HIP;
    for (int s = 0; s < kv->d.n_seq; s++) kv->h_len[s] += tok_off[s + 1] - tok_off[s];
    return TS_OK;
}

int ts_attn_prompt_workspace(int32_t dtype, int32_t n_rows, int32_t n_head_kv, int32_t head_dim, uint64_t *bytes) {
    if (!bytes || !dtype_ok(dtype) || n_rows < 0 || n_head_kv <= 0 || n_head_kv > 65536 || head_dim <= 0 || head_dim % 8 != 0)
        return TS_ERR_INVALID;
    if (head_dim > 256) return TS_ERR_UNSUPPORTED;
    *bytes = prompt_workspace(dtype, n_rows, n_head_kv, head_dim);
    return TS_OK;
}

int ts_attn_prompt(int32_t dtype, const void *d_q, int64_t q_stride, const void *d_k, int64_t k_stride, const void *d_v,
                   int64_t v_stride, const int32_t *tok_off, int32_t n_seq, int32_t n_head, int32_t n_head_kv,
                   int32_t head_dim, float softcap, void *d_out, int64_t out_stride, void *d_workspace,
                   uint64_t workspace_bytes, void *stream) {
    if (!dtype_ok(dtype) || n_seq < 0 || n_head_kv <= 0 || n_head <= 0 || n_head > 65536 || n_head % n_head_kv != 0 ||
        head_dim <= 0 || head_dim % 8 != 0 || !(softcap >= 0.0f) || !std::isfinite(softcap) || !offsets_ok(tok_off, n_seq))
        return TS_ERR_INVALID;
    if (head_dim > 256) return TS_ERR_UNSUPPORTED;
    const int64_t rows = (int64_t)tok_off[n_seq] - tok_off[0];
    if (rows == 0) return TS_OK;
    if (rows * (n_head / n_head_kv) > INT32_MAX - 256) return TS_ERR_INVALID;  // (columns are 32-bit numbers)
    const int64_t qrow = (int64_t)n_head * head_dim, krow = (int64_t)n_head_kv * head_dim;
    if (!rows_ok(d_q, q_stride, qrow, dtype) || !rows_ok(d_k, k_stride, krow, dtype) || !rows_ok(d_v, v_stride, krow, dtype) ||
        !rows_ok(d_out, out_stride, qrow, dtype) || std::max(std::max(q_stride, k_stride), v_stride) > (1 << 22))
        return TS_ERR_INVALID;  // (offsets inside a tile of rows are 32-bit numbers)
    // a token's rows are read by the workgroups of later tokens: the output is apart from all inputs
    const int size = dtype_size(dtype);
    auto span = [&](const void *p, int64_t stride, int64_t row, int end) {
        return (uintptr_t)p + (uintptr_t)((end ? (tok_off[n_seq] - 1) * stride + row : tok_off[0] * stride) * size);
    };
    const uintptr_t o0 = span(d_out, out_stride, qrow, 0), o1 = span(d_out, out_stride, qrow, 1);
    auto apart = [&](const void *p, int64_t stride, int64_t row) { return span(p, stride, row, 1) <= o0 || o1 <= span(p, stride, row, 0); };
    if (!apart(d_q, q_stride, qrow) || !apart(d_k, k_stride, krow) || !apart(d_v, v_stride, krow)) return TS_ERR_INVALID;
    const uint64_t need = prompt_workspace(dtype, rows, n_head_kv, head_dim);
    if (need > 0 && (!d_workspace || workspace_bytes < need)) return TS_ERR_WORKSPACE;
    if (need > 0 && !aligned16(d_workspace)) return TS_ERR_INVALID;
    auto in_ws = [&](const void *p, int64_t stride, int64_t row) {
        const uintptr_t at = span(p, stride, row, 0);
        return need > 0 && bytes_overlap(d_workspace, need, (const void *)at, span(p, stride, row, 1) - at);
    };
    if (in_ws(d_q, q_stride, qrow) || in_ws(d_k, k_stride, krow) || in_ws(d_v, v_stride, krow) || in_ws(d_out, out_stride, qrow))
        return TS_ERR_INVALID;
    PromptCall c;
    c.dtype = dtype;
    c.q = d_q;
    c.k = d_k;
    c.v = d_v;
    c.out = d_out;
    c.q_stride = q_stride;
    c.k_stride = k_stride;
    c.v_stride = v_stride;
    c.out_stride = out_stride;
    c.off = tok_off;
    c.n_seq = n_seq;
    c.n_head = n_head;
    c.n_kv = n_head_kv;
    c.hd = head_dim;
    c.softcap = softcap;
    c.ws = d_workspace;
    return hip_status(launch_prompt(c, as_stream(stream)));
}

// Partials of a call: the prefix's pieces (and one of the own keys for a chunk), then the decode
// kernel's.
static uint64_t shared_part_floats(const ts_kv *kv, int32_t n_head, int32_t n_tok, int slots) {
    return (uint64_t)kv->d.n_seq * n_tok * n_head * slots * (kv->hdp + 2);
}

static bool shared_shape_ok(const ts_kv *kv, const ts_kv *prefix, int32_t n_head, int32_t n_tok) {
    return kv && prefix && kv != prefix && heads_ok(kv, n_head) && n_head <= 65536 && n_tok >= 0 &&
           (int64_t)kv->d.n_seq * n_tok * n_head <= INT32_MAX && kv->d.n_head_kv == prefix->d.n_head_kv &&
           kv->d.head_dim == prefix->d.head_dim && kv->device == prefix->device;
}

int ts_attn_shared_workspace(const ts_kv *kv, const ts_kv *prefix, int32_t n_head, int32_t n_tok, uint64_t *bytes) {
    if (!bytes || !shared_shape_ok(kv, prefix, n_head, n_tok)) return TS_ERR_INVALID;
    *bytes = 0;
    if (n_tok == 0) return TS_OK;
    const int cap = shared_slots_cap(kv->d.n_seq, n_tok, n_head / kv->d.n_head_kv, kv->d.n_head_kv, prefix->d.max_seq,
                                     kv->d.max_seq, kv->n_cu);
    uint64_t n = shared_part_floats(kv, n_head, n_tok, cap) * sizeof(float);
    if (n_tok == 1) {
        uint64_t own;
        ts_attn_decode_workspace(kv, n_head, &own);
        n += own;
    }
    *bytes = n;
    return TS_OK;
}

int ts_attn_shared(ts_kv *kv, const ts_kv *prefix, int32_t prefix_seq, int32_t layer, const float *d_k, const float *d_v,
                   const float *d_q, int32_t n_head, int32_t n_tok, const ts_rope *rope, float softcap, float *d_out,
                   void *d_workspace, uint64_t workspace_bytes, void *stream) {
    if (!shared_shape_ok(kv, prefix, n_head, n_tok) || layer < 0 || layer >= kv->d.n_layers || layer >= prefix->d.n_layers ||
        prefix_seq < 0 || prefix_seq >= prefix->d.n_seq || !(softcap >= 0.0f) || !std::isfinite(softcap) ||
        (d_k == nullptr) != (d_v == nullptr) || (d_k && n_tok != 1) || !aligned16(d_k) || !aligned16(d_v))
        return TS_ERR_INVALID;
    if (n_tok == 0) return TS_OK;
    if (!d_q || !d_out || !aligned16(d_q) || !aligned16(d_out)) return TS_ERR_INVALID;
    // a workgroup reads its rows of q before it writes them, but not before others write theirs
    const uint64_t q_bytes = (uint64_t)kv->d.n_seq * n_tok * n_head * kv->d.head_dim * sizeof(float);
    if (d_out != d_q && bytes_overlap(d_q, q_bytes, d_out, q_bytes)) return TS_ERR_INVALID;
    // the own positions continue the prefix's: slot p of a sequence is position window base + p (of all its
    // slots: no sinks), and the prefix ends at its length plus its own window base
    const int P = prefix->h_len[prefix_seq];
    const int64_t end = P > 0 ? (int64_t)P + prefix->h_rot[prefix_seq] : 0;
    for (int s = 0; s < kv->d.n_seq; s++) {
        if (kv->h_rot[s] < end || (P > 0 && kv->h_sink[s] != 0)) return TS_ERR_INVALID;
        if ((int64_t)kv->h_len[s] + n_tok > kv->d.max_seq) return TS_ERR_OVERFLOW;
    }
    const int rc = check_rope(rope, kv->d.head_dim, rot_end(kv, n_tok));
    if (rc) return rc;
    if (P == 0)
        return n_tok > 1 ? ts_attn_prefill(kv, layer, d_q, n_head, n_tok, rope, softcap, d_out, stream)
               : d_k     ? ts_attn_decode_append(kv, layer, d_k, d_v, d_q, n_head, rope, softcap, d_out, d_workspace,
                                                 workspace_bytes, stream)
                         : ts_attn_decode(kv, layer, d_q, n_head, rope, softcap, d_out, d_workspace, workspace_bytes, stream);
    uint64_t need;
    ts_attn_shared_workspace(kv, prefix, n_head, n_tok, &need);
    if (need > 0 && (!d_workspace || workspace_bytes < need)) return TS_ERR_WORKSPACE;
    if (need > 0 && !aligned16(d_workspace)) return TS_ERR_INVALID;
    const uint64_t kv_bytes = q_bytes / n_head * kv->d.n_head_kv;
    if (bytes_overlap(d_workspace, need, d_q, q_bytes) || bytes_overlap(d_workspace, need, d_out, q_bytes) ||
        bytes_overlap(d_workspace, need, d_k, kv_bytes) || bytes_overlap(d_workspace, need, d_v, kv_bytes))
        return TS_ERR_INVALID;

    SharedCall c;
    c.own = rotating_layer(kv, layer, rope, stream);
    c.pre = prefix->layer(layer);
    c.prefix_seq = prefix_seq;
    c.prefix_len = P;
    c.d_len = kv->d_len;
    c.q = d_q;
    c.n_head = n_head;
    c.n_tok = n_tok;
    c.rope = rope->d_table;
    c.rope_pairs = rope->rope_dim / 2;
    c.rope_rows = rope->n_pos;
    c.softcap = softcap;
    c.out = d_out;
    const int G = n_head / kv->d.n_head_kv;
    const int own_max = *std::max_element(kv->h_len.begin(), kv->h_len.end()) + n_tok;
    c.plan = shared_plan(kv->d.n_seq, n_tok, G, kv->d.n_head_kv, P, own_max, kv->n_cu);
    c.part = static_cast<float *>(d_workspace);
    c.own_part = nullptr;
    c.own_chunk = c.own_split = 1;
    c.hlen = -1;
    c.k_new = d_k;
    c.v_new = d_v;
    c.n_cu = kv->n_cu;
    if (n_tok == 1) {
        c.own_part = c.part + shared_part_floats(kv, n_head, 1, c.plan.n_part);
        for (int s = 0; s < kv->d.n_seq; s++) kv->h_ctx[s] = kv->h_len[s] + 1;
        shared_own_plan(kv->h_ctx.data(), kv->d.n_seq, kv->d.n_head_kv, G, kv->n_cu, &c.own_chunk, &c.own_split);
        // (an eager call gives a lone sequence's length with the launch, as ts_attn_decode)
        if (kv->d.n_seq == 1 && !capturing(stream) && !kv->len_captured) c.hlen = kv->h_len[0];
    }
    return hip_status(launch_shared(c, as_stream(stream)));
}

}  // extern "C"
