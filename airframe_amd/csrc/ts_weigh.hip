// ts_weigh.hip -- what every cached slot receives of the attention of new tokens, for gfx950.
//
// For the new tokens t and query heads h of one kv head, P[t,h,p] = softmax over the slots p the token
// sees: w[p] = (w[p]) + sum over t and h of P[t,h,p].  The sums over columns need each softmax's final
// reference and sum, so they come behind the attention itself.
#include "ts_evict.h"
#include "ts_mfma.h"

namespace ts {
namespace {

struct WeighArgs {
    KvLayerView L;
    const int32_t *len;
    const float *q, *rope;
    int rope_pairs, rope_rows, n_head, G, n_tok;
    float inv_sqrt_hd, softcap;
    int max_seq;
    float *w;
    bool fresh;
    float *qr, *lse;  // rotated q [rows][HD], the softmax's log2 sum [rows]
};

// q rows normalized, rotated and scaled.
template <int HD>
__global__ __launch_bounds__(64) void weigh_q_kernel(WeighArgs a) {
    const int row = blockIdx.x, lane = threadIdx.x, hdr = a.L.hdr;
    const int tok = row / a.n_head % a.n_tok, s = row / a.n_head / a.n_tok;
    const float *q = a.q + (size_t)row * hdr;
    const float ns = a.L.qn ? qk_norm_scale(q, hdr, a.L.norm_eps) : 1.0f;
    const int pos = min(rot_of(a.L, s, a.len[s] + tok), a.rope_rows - 1);
    const float mul = a.softcap > 0.0f ? a.inv_sqrt_hd : a.inv_sqrt_hd * kLog2e;
    for (int i = lane; i < HD / 2; i += 64) {
        float x0 = 0.0f, x1 = 0.0f;
        if (2 * i < hdr) {
            x0 = q[2 * i];
            x1 = q[2 * i + 1];
            if (a.L.qn) {
                x0 = qk_norm_apply(x0, ns, a.L.qn[2 * i]);
                x1 = qk_norm_apply(x1, ns, a.L.qn[2 * i + 1]);
            }
            if (i < a.rope_pairs)
                rope_rotate(x0, x1, *reinterpret_cast<const float2 *>(a.rope + ((size_t)pos * a.rope_pairs + i) * 2));
        }
        a.qr[(size_t)row * HD + 2 * i] = x0 * mul;
        a.qr[(size_t)row * HD + 2 * i + 1] = x1 * mul;
    }
}

// Score of slot p for a rotated q row, in the exp2 domain.
template <int HD>
__device__ inline float score(const WeighArgs &a, size_t st, int p, const float *q) {
    const uint32_t *k = reinterpret_cast<const uint32_t *>(a.L.kp + st * a.L.P * (HD / 2));
    float dot = 0.0f;
    for (int u = 0; u < HD / 8; u++) {
        const uint32_t w = k[k_word_idx<HD>(p, u)];
#pragma unroll
        for (int e = 0; e < 8; e++) dot += (float)((int)(w >> (4 * e) & 15) - 8) * q[8 * u + e];
    }
    float x = dot * a.L.ks[st * a.L.P + p];
    if (a.softcap > 0.0f) x = tanhf(x / a.softcap) * a.softcap * kLog2e;
    return x;
}

template <int HD>
__global__ __launch_bounds__(256) void weigh_stats_kernel(WeighArgs a) {
    __shared__ float q[HD], ms[4], ls[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    const int head = row % a.n_head, tok = row / a.n_head % a.n_tok, s = row / a.n_head / a.n_tok;
    const size_t st = (size_t)s * a.L.H + head / a.G;
    for (int i = tid; i < HD; i += 256) q[i] = a.qr[(size_t)row * HD + i];
    __syncthreads();
    const int n = min(a.len[s] + tok + 1, a.L.P);
    float m = kMinit, l = 0.0f;
    for (int p = tid; p < n; p += 256) {
        const float x = score<HD>(a, st, p, q), mn = fmaxf(m, x);
        l = l * exp2f(m - mn) + exp2f(x - mn);
        m = mn;
    }
    const float M = wave_max(m);
    l = wave_sum(l * exp2f(m - M));
    if ((tid & 63) == 0) {
        ms[tid >> 6] = M;
        ls[tid >> 6] = l;
    }
    __syncthreads();
    if (tid == 0) {
        float mm = kMinit, ll = 0.0f;
        for (int i = 0; i < 4; i++) mm = fmaxf(mm, ms[i]);
        for (int i = 0; i < 4; i++) ll += ls[i] * exp2f(ms[i] - mm);
        a.lse[row] = mm + log2f(ll);
    }
}

template <int HD>
__global__ __launch_bounds__(256) void weigh_sum_kernel(WeighArgs a) {
    const int p = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, s = blockIdx.z;
    const size_t st = (size_t)s * a.L.H + h;
    const int len = a.len[s], n = len + a.n_tok;
    if (p >= a.max_seq || len + a.n_tok > a.max_seq) return;  // (a graph replayed past the capacity)
    float *w = a.w + st * a.max_seq + p;
    if (p >= n) {
        if (a.fresh) *w = 0.0f;
        return;
    }
    float sum = 0.0f;
    for (int t = max(0, p - len); t < a.n_tok; t++)
        for (int g = 0; g < a.G; g++) {
            const size_t row = ((size_t)s * a.n_tok + t) * a.n_head + h * a.G + g;
            sum += exp2f(score<HD>(a, st, p, a.qr + row * HD) - a.lse[row]);
        }
    *w = a.fresh ? sum : *w + sum;
}

}  // namespace

uint64_t weigh_workspace(int n_seq, int n_tok, int n_head, int stored_hd) {
    return (uint64_t)n_seq * n_tok * n_head * (stored_hd + 1) * sizeof(float);
}

hipError_t launch_weigh(const WeighCall &c, hipStream_t st) {
    WeighArgs a;
    a.L = c.L;
    a.len = c.d_len;
    a.q = c.q;
    a.rope = c.rope;
    a.rope_pairs = c.rope_pairs;
    a.rope_rows = c.rope_rows;
    a.n_head = c.n_head;
    a.G = c.n_head / c.L.H;
    a.n_tok = c.n_tok;
    a.inv_sqrt_hd = 1.0f / sqrtf((float)c.L.hdr);
    a.softcap = c.softcap;
    a.max_seq = c.max_seq;
    a.w = c.w;
    a.fresh = c.fresh;
    const int rows = c.L.S * c.n_tok * c.n_head;
    a.qr = c.ws;
    a.lse = c.ws + (size_t)rows * c.L.hd;
    const dim3 grid((c.max_seq + 255) / 256, c.L.H, c.L.S);
#define TS_WEIGH(HDV)                                   \
    {                                                   \
        weigh_q_kernel<HDV><<<rows, 64, 0, st>>>(a);     \
        weigh_stats_kernel<HDV><<<rows, 256, 0, st>>>(a); \
        weigh_sum_kernel<HDV><<<grid, 256, 0, st>>>(a);  \
    }
    if (c.L.hd == 256) TS_WEIGH(256)
    else if (c.L.hd == 128) TS_WEIGH(128)
    else TS_WEIGH(64)
#undef TS_WEIGH
    return hipGetLastError();
}

}  // namespace ts
