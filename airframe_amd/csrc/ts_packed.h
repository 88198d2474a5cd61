// ts_packed.h -- packed batches: the rows of all sequences one after another, sequence s owning
// rows tok[s] .. tok[s+1].  The offsets are host numbers: the ABI checks them there, and the
// kernels get them by value with the launch, so that a captured call holds its own copy and
// no call waits for an upload.  One launch takes up to kPackSeqs sequences (the argument segment
// holds 4 KB); longer batches take several.
#pragma once
#include "ts_internal.h"

namespace ts {

constexpr int kPackSeqs = 128;

// Sequences seq0 .. seq0 + n - 1 of a batch: their first rows, and the first work item (a block of
// positions, a tile of columns) of each; entry n closes both.  pos0: a position per sequence.
struct PackTable {
    int32_t n, seq0;
    int32_t tok[kPackSeqs + 1];
    int32_t item[kPackSeqs + 1];
    int32_t pos0[kPackSeqs];
};

// Fills t with the sequences from seq0 on (items(rows) work items each; pos0 null: zeros) and
// returns how many it took.
template <class F>
inline int pack_fill(PackTable &t, const int32_t *off, const int32_t *pos0, int n_seq, int seq0, F items) {
    t.seq0 = seq0;
    t.n = std::min(n_seq - seq0, kPackSeqs);
    t.tok[0] = off[seq0];
    t.item[0] = 0;
    for (int i = 0; i < t.n; i++) {
        t.tok[i + 1] = off[seq0 + i + 1];
        t.item[i + 1] = t.item[i] + items(off[seq0 + i + 1] - off[seq0 + i]);
        t.pos0[i] = pos0 ? pos0[seq0 + i] : 0;
    }
    return t.n;
}

// Offsets that can be used: no row before the first, none of negative length.
inline bool offsets_ok(const int32_t *off, int n_seq) {
    if (!off || off[0] < 0) return false;
    for (int s = 0; s < n_seq; s++)
        if (off[s + 1] < off[s]) return false;
    return true;
}

inline int dtype_size(int32_t dtype) { return dtype == TS_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t dtype) { return dtype == TS_DTYPE_F32 || dtype == TS_DTYPE_F16 || dtype == TS_DTYPE_BF16; }

#if defined(__HIPCC__)
// The entry whose items hold item b (the last one that starts at or before it): every lane
// compares its entries, so the search is one round of loads and not a chain of them.
__device__ inline int pack_find(const PackTable &t, int b) {
    const int lane = __lane_id();
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPackSeqs; i += 64)
        c += __popcll(__builtin_amdgcn_ballot_w64(i + lane < t.n && t.item[i + lane] <= b));
    return __builtin_amdgcn_readfirstlane(c - 1);
}

// 8 consecutive elements of a row as f32 (16-byte aligned).
__device__ inline void load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ inline void load8(const _Float16 *p, float (&x)[8]) {
    const f16x8 v = *reinterpret_cast<const f16x8 *>(p);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)v[e];
}
__device__ inline void load8(const __bf16 *p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    }
}
// The same back, each rounded once (nearest even).
__device__ inline void store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ inline void store8(_Float16 *p, const float (&x)[8]) {
    f16x8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (_Float16)x[e];
    *reinterpret_cast<f16x8 *>(p) = v;
}
__device__ inline void store8(__bf16 *p, const float (&x)[8]) {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (__bf16)x[e];
    *reinterpret_cast<bf16x8 *>(p) = v;
}
#endif

// Launchers of ts_packed.hip.
hipError_t launch_rope_table(float *table, int32_t n_pos, int32_t rope_dim, double base, double factor, double l_train,
                             double alpha, double beta, double mult, hipStream_t st);
hipError_t launch_rope_apply(int32_t dtype, int32_t layout, const void *x, int64_t x_stride, const int32_t *pos, int n_tok,
                             int n_head, int hd, const float *table, int pairs, int n_pos, void *out, int64_t out_stride,
                             hipStream_t st);
hipError_t launch_append_packed(const KvLayerView &L, const int32_t *d_len, int32_t dtype, const void *k, int64_t k_stride,
                                const void *v, int64_t v_stride, const int32_t *off, const float *rope, int32_t rope_pairs,
                                int32_t n_pos, hipStream_t st);
hipError_t launch_read_packed(const KvLayerView &L, const int32_t *pos0, const int32_t *off, int32_t dtype, void *k,
                              int64_t k_stride, void *v, int64_t v_stride, hipStream_t st);
hipError_t launch_len_add(int32_t *d_len, int n_seq, const int32_t *off, hipStream_t st);

}  // namespace ts
