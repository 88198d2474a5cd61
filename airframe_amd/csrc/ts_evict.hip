// ts_evict.hip -- eviction from the INT4 cache, for gfx950: which slots stay, by the attention they have
// received, and their rows moved together.
#include "ts_evict.h"

namespace ts {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- the choice ----------------------------------------------------------------------------------
//
// A row (one layer, sequence and kv head) keeps its first n_sink slots, its last n_recent, and of those
// between the `need` largest weights, equal ones from the lowest slot on.  Weights are compared as
// unsigned keys in their order (-0 as 0, NaN above all).

__device__ inline uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (u == 0x80000000u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 256;

__device__ inline int block_sum(int v, int *s, int tid) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((tid & 63) == 0) s[tid >> 6] = v;
    __syncthreads();
    int sum = 0;
    for (int i = 0; i < kSelThreads / 64; i++) sum += s[i];
    return sum;
}

__global__ __launch_bounds__(kSelThreads) void select_kernel(const float *w, const int32_t *len, int n_seq, int H, int max_seq,
                                                             int keep, int n_sink, int n_recent, int32_t *slots) {
    __shared__ int s_sum[kSelThreads / 64], s_gt[kSelThreads / 64], s_eq[kSelThreads / 64];
    const size_t row = blockIdx.x;
    const int s = (int)(row / H % n_seq), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(len[s], max_seq);
    w += row * max_seq;
    slots += row * keep;
    if (n <= keep) {
        for (int j = tid; j < keep; j += kSelThreads) slots[j] = j < n ? j : -1;
        return;
    }
    const int lo = n_sink, hi = n - n_recent, need = keep - n_sink - n_recent;
    // the need-th largest key: its bits from the highest down
    uint32_t t = 0;
    for (int b = 31; b >= 0 && need > 0; b--) {
        const uint32_t c = t | 1u << b;
        int cnt = 0;
        for (int p = lo + tid; p < hi; p += kSelThreads) cnt += order_key(w[p]) >= c;
        if (block_sum(cnt, s_sum, tid) >= need) t = c;
    }
    int above = 0;
    for (int p = lo + tid; p < hi; p += kSelThreads) above += order_key(w[p]) > t;
    const int ties = need > 0 ? need - block_sum(above, s_sum, tid) : 0;  // of those equal to it
    int out = 0, eq = 0;
    for (int p0 = 0; p0 < n; p0 += kSelThreads) {
        const int p = p0 + tid;
        const bool mid = p >= lo && p < hi;
        const uint32_t k = mid && need > 0 ? order_key(w[p]) : 0;
        const bool is_eq = mid && need > 0 && k == t, sure = p < n && (!mid || (need > 0 && k > t));
        const uint64_t beq = __ballot(is_eq);
        __syncthreads();
        if (lane == 0) s_eq[wave] = __popcll(beq);
        __syncthreads();
        int rank = eq + __popcll(beq & ((1ull << lane) - 1));
        for (int i = 0; i < wave; i++) rank += s_eq[i];
        const bool take = sure || (is_eq && rank < ties);
        const uint64_t bt = __ballot(take);
        if (lane == 0) s_gt[wave] = __popcll(bt);
        __syncthreads();
        int at = out + __popcll(bt & ((1ull << lane) - 1));
        for (int i = 0; i < wave; i++) at += s_gt[i];
        if (take && at < keep) slots[at] = p;
        for (int i = 0; i < kSelThreads / 64; i++) {
            out += s_gt[i];
            eq += s_eq[i];
        }
    }
}

// ---- the rows ------------------------------------------------------------------------------------
//
// Slots are ascending, so a row never moves up: the source of slot j is j or a later one.  One wave
// takes one slice of the rows of one (layer, sequence, kv head) and walks the slots in windows of 64:
// it reads a window's sources before it writes the window, and no later window reads a slot that an
// earlier one has written, so the move needs no second copy, also in place.  Slices: the K words of
// each lane group g, 16-byte chunks of V's lane groups, the scales with the weights.

template <int HD>
constexpr int kKeepSlices = 4 + HD / 64 + 1;

template <int HD>
__global__ __launch_bounds__(64) void keep_kernel(KeepCall a) {
    const unsigned slice = blockIdx.x % kKeepSlices<HD>, row = blockIdx.x / kKeepSlices<HD>;
    const int lane = threadIdx.x, H = a.src.H;
    const int h = row % H, i = row / H % a.n_seq, layer = row / H / a.n_seq;
    const int len = min(a.src_len[a.src_seq + i], a.src_max), n = min(len, a.keep);
    const size_t srow = (size_t)(a.src_seq + i) * H + h, drow = (size_t)(a.dst_seq + i) * H + h;
    const int sP = a.src.P, dP = a.dst.P;
    const int32_t *slots = a.slots + (size_t)row * a.slot_row;
    const size_t so = a.src_layer * layer, dof = a.dst_layer * layer;
    // (a slot outside the source reads one inside it)
    auto source = [&](int j) { return j < n ? min(max(slots[j], 0), len - 1) : 0; };
    if (slice < 4) {
        constexpr int W = HD / 32;  // words of a slot in lane group g
        const int g = slice;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(a.src.kp + so + srow * sP * (HD / 2));
        uint32_t *dst = reinterpret_cast<uint32_t *>(a.dst.kp + dof + drow * dP * (HD / 2));
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane, p = source(j);
            uint32_t x[W];
#pragma unroll
            for (int e = 0; e < W; e++) x[e] = src[k_word_idx<HD>(p, 8 * (e >> 1) + 2 * g + (e & 1))];
            if (j < n) {
#pragma unroll
                for (int e = 0; e < W; e++) dst[k_word_idx<HD>(j, 8 * (e >> 1) + 2 * g + (e & 1))] = x[e];
            }
        }
    } else if (slice < 4 + HD / 64) {
        const int td4 = slice - 4;
        const u32x4 *src = reinterpret_cast<const u32x4 *>(a.src.vp + so + srow * (sP / 32) * (HD * 16));
        u32x4 *dst = reinterpret_cast<u32x4 *>(a.dst.vp + dof + drow * (dP / 32) * (HD * 16));
        const int g = lane >> 4, dl = lane & 15;
        for (int j0 = 0; j0 < n; j0 += 32) {
            const int mine = source(j0 + (lane & 31));
            u32x4 x = {0, 0, 0, 0};
            uint32_t left = 0;  // nibbles of slots from n on stay
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int jj = (e < 4 ? 0 : 16) + 4 * g + (e & 3);
                const int p = __shfl(mine, jj, 64), r = p & 31;
                const u32x4 w = src[(size_t)(p >> 5) * HD + td4 * 64 + 16 * ((r & 15) >> 2) + dl];
                const int sh = 4 * ((r & 3) + 4 * (r >> 4));
                if (j0 + jj < n) {
#pragma unroll
                    for (int c = 0; c < 4; c++) x[c] |= (w[c] >> sh & 15) << (4 * e);
                } else {
                    left |= 15u << (4 * e);
                }
            }
            u32x4 *to = dst + (size_t)(j0 >> 5) * HD + td4 * 64 + lane;
            if (left) {
                const u32x4 old = *to;
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] = (x[c] & ~left) | (old[c] & left);
            }
            *to = x;
        }
    } else {
        const float *ks = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(a.src.ks) + so) + srow * sP;
        const float *vs = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(a.src.vs) + so) + srow * sP;
        float *kd = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(a.dst.ks) + dof) + drow * dP;
        float *vd = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(a.dst.vs) + dof) + drow * dP;
        const float *ws = a.src_w ? a.src_w + ((size_t)layer * a.src.S * H + srow) * a.src_max : nullptr;
        float *wd = a.dst_w ? a.dst_w + ((size_t)layer * a.dst.S * H + drow) * a.dst_max : nullptr;
        for (int j0 = 0; j0 < n; j0 += 64) {
            const int j = j0 + lane, p = source(j);
            const float k = ks[p], v = vs[p], w = wd ? ws[p] : 0.0f;
            if (j < n) {
                kd[j] = k;
                vd[j] = v;
                if (wd) wd[j] = w;
            }
        }
        // slots behind the kept ones have received nothing
        const int end = a.in_place ? len : a.dst_max;
        if (wd)
            for (int j = n + lane; j < end; j += 64) wd[j] = 0.0f;
    }
}

__global__ void keep_len_kernel(KeepCall a) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.n_seq) return;
    const int len = min(a.src_len[a.src_seq + i], a.src_max), n = min(len, a.keep), rot = a.src_rot[a.src_seq + i];
    a.dst_len[a.dst_seq + i] = n;
    a.dst_rot[a.dst_seq + i] = rot + len - n;
    a.dst_sink[a.dst_seq + i] = 0;
}

}  // namespace

hipError_t launch_select(const float *w, const int32_t *d_len, int n_layers, int n_seq, int H, int max_seq, int keep,
                         int n_sink, int n_recent, int32_t *d_slots, hipStream_t st) {
    select_kernel<<<(unsigned)(n_layers * n_seq * H), kSelThreads, 0, st>>>(w, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, d_slots);
    return hipGetLastError();
}

hipError_t launch_keep(const KeepCall &c, hipStream_t st) {
    const unsigned rows = (unsigned)(c.n_layers * c.n_seq * c.src.H);
    if (c.src.hd == 256) keep_kernel<256><<<rows * kKeepSlices<256>, 64, 0, st>>>(c);
    else if (c.src.hd == 128) keep_kernel<128><<<rows * kKeepSlices<128>, 64, 0, st>>>(c);
    else keep_kernel<64><<<rows * kKeepSlices<64>, 64, 0, st>>>(c);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    keep_len_kernel<<<(c.n_seq + 63) / 64, 64, 0, st>>>(c);
    return hipGetLastError();
}

}  // namespace ts
