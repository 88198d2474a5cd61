// ts_host.h -- checks and conversions shared by the host files of the C ABI.
#pragma once
#include "ts_internal.h"

namespace ts {

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

// True when work enqueued on the stream now goes into a graph being captured.
inline bool capturing(void *stream) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(as_stream(stream), &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}

// A call that changes the device lengths: note when it is being captured.
inline void note_len_change(ts_kv *kv, void *stream) {
    if (capturing(stream)) kv->len_captured = true;
}

inline int hip_status(hipError_t e) { return e == hipSuccess ? TS_OK : TS_ERR_HIP; }

// The kernels move rows in 16-byte pieces.
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// Largest rotation position (exclusive) the next n_tok tokens of any sequence use: slots past
// the sinks are rotated at slot + window base.
inline int64_t rot_end(const ts_kv *kv, int32_t n_tok) {
    int64_t m = 0;
    for (int s = 0; s < kv->d.n_seq; s++) m = std::max<int64_t>(m, (int64_t)kv->h_len[s] + kv->h_rot[s] + n_tok);
    return m;
}

inline int check_rope(const ts_rope *rope, int hd, int64_t max_pos_exclusive) {
    if (!rope) return TS_ERR_INVALID;
    if (rope->rope_dim > hd) return TS_ERR_INVALID;
    if (max_pos_exclusive > rope->n_pos) return TS_ERR_INVALID;
    return TS_OK;
}

// Any GQA group size: the decode takes more than 8 query heads per kv head as several head
// groups (each reads the kv head's stream).
inline bool heads_ok(const ts_kv *kv, int32_t n_head) { return n_head > 0 && n_head % kv->d.n_head_kv == 0; }

}  // namespace ts
