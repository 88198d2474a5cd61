// ts_weigh_token.hip -- one token's attention over the INT4 cache that adds up what every slot receives, for
// gfx950.
//
// A slot's probability needs the final reference and sum of its head's softmax, which no split of the keys has.
// The decode kernels therefore leave every score beside their partials (4 bytes per query head and slot; the cached
// row behind it has hd + 8 per kv head).  A workgroup that holds all slots of its kv head turns them into sums itself,
// from L2; otherwise one more launch joins the partials and does:
//   w[p] = (w[p]) + sum over the query heads g of one kv head of 2^(x_g[p] - lse_g),
//   lse = M + log2(sum over the splits of 2^(m - M) l).
// In the kernel where no sequence is split: 32 sequences of 4096-8192 slots, 32 heads over 8 of 128 dims 56 us (61 with a
// launch for the sums; 210 MB, 3.8 TB/s), one of 511 slots of 64 dims 9.5 us (12.4; a chain of round trips).  8 of
// 1001-16003: 21.4 us the splits, 6.1 the join and sums; 4 of 700-6001 with 256 dims 15.6 and 4.0.
#include <cfloat>

#include "ts_decode_int.h"
#include "ts_evict.h"

namespace ts {
namespace {

template <int HD, bool SOFTCAP, bool NORM, bool PAD, int NW>
__global__ __launch_bounds__(64 * NW, NW > 4 ? 1 : (HD > 128 ? 1 : 2)) void weigh_split_kernel(DecodeArgs a) {
#define TS_SPLIT_X blockIdx.x
#define TS_SPLIT_Y blockIdx.y
#define TS_SPLIT_Z blockIdx.z
#define TS_SPLIT_KEEP false
#define TS_SPLIT_SCORES true
#define TS_SPLIT_LDS                                   \
    __shared__ __align__(16) DecodeSplitSmem<HD, NW> sm; \
    __shared__ __align__(16) float kd[HD], vd[HD];       \
    __shared__ float xnew[8], lse_s[8];
#include "ts_decode_split_body.h"
#undef TS_SPLIT_X
#undef TS_SPLIT_Y
#undef TS_SPLIT_Z
#undef TS_SPLIT_LDS
#undef TS_SPLIT_KEEP
#undef TS_SPLIT_SCORES
}

struct SumArgs {
    DecodeArgs d;
    float *w;
    int n_join, n_chunk;  // workgroups that join a head's splits, then n_chunk per (sequence, kv head)
};

constexpr int kSumSlots = 1024;  // slots per workgroup

// Both of a split batch in one launch, which none of the other's results needs: the heads' joins, and kSumSlots slots of a kv
// head per workgroup, whose heads' lse it takes from the splits' stats itself (a round trip, no launch more).
template <int HD>
__global__ __launch_bounds__(256) void weigh_sum_token_kernel(SumArgs a) {
    const DecodeArgs &d = a.d;
    const int tid = threadIdx.x, H = d.L.H;
    if ((int)blockIdx.x < a.n_join) {
        const int head = blockIdx.x % d.n_head, s = blockIdx.x / d.n_head;
        const int n = (d.hlen >= 0 ? d.hlen : d.len[s]) + 1, ns = min((n + d.chunk - 1) / d.chunk, d.n_split);
        if (ns > 1 && n <= d.L.P) combine_rows<HD>(d, head, s, ns, tid);
        return;
    }
    const int b = blockIdx.x - a.n_join, h = b % H, s = b / H % d.L.S, p0 = b / H / d.L.S * kSumSlots;
    const int n = (d.hlen >= 0 ? d.hlen : d.len[s]) + 1;
    float *const w = a.w + ((size_t)s * H + h) * d.max_seq;
    if (n > d.max_seq) return;  // (a graph replayed past the capacity)
    const int ns = min((n + d.chunk - 1) / d.chunk, d.n_split), G = d.Gt;
    extern __shared__ float lse[];  // [G]
    const size_t rows = (size_t)d.L.S * d.n_head * d.n_split, head0 = (size_t)s * d.n_head + h * G;
    if (p0 < n) {
        const int wave = tid >> 6, lane = tid & 63;
        for (int g = wave; g < G; g += 4) {
            const float *m = d.ws + rows * HD + (head0 + g) * d.n_split, *l = m + rows;
            float M = kMinit, sum = 0.0f;
            for (int i = lane; i < ns; i += 64) M = fmaxf(M, m[i]);
            M = wave_max(M);
            for (int i = lane; i < ns; i += 64) sum += __builtin_amdgcn_exp2f(m[i] - M) * l[i];
            sum = wave_sum(sum);
            if (lane == 0) lse[g] = M + __log2f(sum);
        }
    }
    __syncthreads();
    const float *x = d.scores + head0 * d.L.P;
    const int p = p0 + 4 * tid;
    if (p >= (d.fresh ? d.max_seq : n)) return;
    if (G <= 8) return sum_scores<8, 1>(d, x, w, G, n, lse, p, 0);
    floatx4 sum = (floatx4)0.0f;
    if (p < n)
        for (int g = 0; g < G; g++) {
            const floatx4 v = *reinterpret_cast<const floatx4 *>(x + (size_t)g * d.L.P + p);
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += __builtin_amdgcn_exp2f(v[e] - lse[g]);
        }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (p + e < n) w[p + e] = d.fresh ? sum[e] : w[p + e] + sum[e];
        else if (d.fresh && p + e < d.max_seq) w[p + e] = 0.0f;
    }
}

template <int HD, bool SC, bool NM, bool PAD>
void launch_16x16_pad(const DecodeArgs &a, dim3 grid, int nw, hipStream_t st) {
    if (HD <= 128 && nw == 8)
        weigh_split_kernel<HD, SC, NM, PAD, HD <= 128 ? 8 : 4><<<grid, 64 * 8, 0, st>>>(a);
    else if (HD <= 64 && nw == 16)
        weigh_split_kernel<HD, SC, NM, PAD, HD <= 64 ? 16 : 4><<<grid, 64 * 16, 0, st>>>(a);
    else
        weigh_split_kernel<HD, SC, NM, PAD, 4><<<grid, 64 * 4, 0, st>>>(a);
}

template <int HD, bool SC, bool NM>
void launch_scores(const DecodeArgs &a, const DecodePlan &plan, hipStream_t st) {
    const bool pad = a.L.hdr != a.L.hd;
    const dim3 grid(plan.n_split, a.L.H * a.NG, a.L.S);
    if (plan.g4) launch_integer<HD, SC, NM, true>(a, plan.n_split, pad, a.Gt, st);
    else if (pad) launch_16x16_pad<HD, SC, NM, true>(a, grid, plan.nw, st);
    else launch_16x16_pad<HD, SC, NM, false>(a, grid, plan.nw, st);
}

template <int HD>
void launch_token(const SumArgs &a, const DecodePlan &plan, unsigned blocks, hipStream_t st) {
    const bool cap = a.d.softcap > 0.0f, norm = a.d.L.qn != nullptr || a.d.L.kn != nullptr;
    if (cap) norm ? launch_scores<HD, true, true>(a.d, plan, st) : launch_scores<HD, true, false>(a.d, plan, st);
    else norm ? launch_scores<HD, false, true>(a.d, plan, st) : launch_scores<HD, false, false>(a.d, plan, st);
    if (!a.d.w) weigh_sum_token_kernel<HD><<<blocks, 256, a.d.Gt * sizeof(float), st>>>(a);
}

uint64_t token_part_floats(int n_seq, int n_head, int n_split, int hd) { return (uint64_t)n_seq * n_head * n_split * (hd + 2); }

}  // namespace

uint64_t weigh_token_workspace(int n_seq, int n_head, int n_kv, int P, int max_seq, int stored_hd, int n_cu) {
    const uint64_t parts = token_part_floats(n_seq, n_head, decode_cap(n_kv, max_seq, n_cu), stored_hd) * sizeof(float);
    return parts + 256 + (uint64_t)n_seq * n_head * P * sizeof(float);
}

hipError_t launch_weigh_token(const WeighCall &c, const DecodePlan &plan, hipStream_t st) {
    SumArgs a;
    DecodeArgs &d = a.d;
    d.L = c.L;
    d.len = c.d_len;
    d.hlen = c.hlen;
    d.q = c.q;
    d.rope = c.rope;
    d.rope_pairs = c.rope_pairs;
    d.n_head = c.n_head;
    d.Gt = c.n_head / c.L.H;
    d.NG = plan.g4 ? 1 : (d.Gt + 7) / 8;
    d.G = plan.g4 ? d.Gt : std::min(d.Gt, 8);
    d.chunk = plan.chunk;
    d.n_split = plan.n_split;
    d.inv_sqrt_hd = 1.0f / sqrtf((float)c.L.hdr);
    d.softcap = c.softcap;
    d.inv_softcap = c.softcap > 0.0f ? std::min(1.0f / c.softcap, FLT_MAX) : 0.0f;
    d.out = c.out;
    d.ws = reinterpret_cast<float *>(c.ws);
    d.k_new = c.k_new;
    d.v_new = c.v_new;
    d.adv_len = d.adv_ctr = nullptr;
    const uint64_t parts = token_part_floats(c.L.S, c.n_head, plan.n_split, c.L.hd) * sizeof(float);
    // (whole cache lines: a head's scores are read back by the workgroup that wrote them, and by no other before)
    d.scores = reinterpret_cast<float *>(((uintptr_t)c.ws + parts + 255) / 256 * 256);
    d.max_seq = c.max_seq;
    d.fresh = c.fresh;
    a.w = c.w;
    // no sequence split, one workgroup for all query heads of a kv head: it adds up itself
    d.w = plan.n_split == 1 && d.NG == 1 ? c.w : nullptr;
    const int slots = c.fresh || c.captured ? c.max_seq : c.own_max;
    a.n_join = plan.n_split > 1 ? c.n_head * c.L.S : 0;
    a.n_chunk = (slots + kSumSlots - 1) / kSumSlots;
    const unsigned blocks = (unsigned)(a.n_join + a.n_chunk * c.L.H * c.L.S);
    if (c.L.hd == 256) launch_token<256>(a, plan, blocks, st);
    else if (c.L.hd == 128) launch_token<128>(a, plan, blocks, st);
    else launch_token<64>(a, plan, blocks, st);
    return hipGetLastError();
}

}  // namespace ts
