// ts_shared.hip -- attention of a batch whose sequences share a prefix, for gfx950.
//
// Every sequence's new tokens attend to the prefix (positions 0 .. P-1, one sequence of another INT4
// cache) and then to its own keys (position P + slot).  A softmax over both is the join of two:
// with o, m, l the unnormalized output, reference and sum over a part of the keys,
//   out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// The prefix's part is one matrix product for the whole batch: all (sequence, token, head) columns of
// a kv head against each window of keys, so the prefix is read and unpacked once per 128 columns
// instead of once per sequence.  Its keys are divided among workgroups until they fill the chip;
// the pieces are joined by a last kernel, with the own keys' parts: of the decode kernel for one
// token, of the same window walk for a chunk.
//
// 32 heads over 8 of 128 dims, 32 sequences of 60 to 500 own keys behind 8192: 29.5 us (shared_kernel 24.4,
// a CU's four windows with the q before and the partials behind them; join 6), of which the bytes would take
// 3.4 and the matrix work 4; the same with the new tokens' append in the launch.  Chunks of 256 tokens of 8 sequences
// behind 4097: 252 to 269 us by card, 142 GFLOP that hi and lo terms of q and P make 240: 0.89 to 0.95 PFLOP/s executed.
#include "ts_shared.h"

#include "ts_decode_split.h"
#include "ts_window.h"

namespace ts {
namespace {

struct SharedArgs {
    KvLayerView own, pre;
    int prefix_seq, prefix_len;
    const int32_t *len;
    const float *q, *rope;
    int rope_pairs, rope_rows, n_head, G, n_tok;
    bool chain;                // one job walks the prefix and then a sequence's own keys
    int n_blk, n_part, chunk;  // the prefix's jobs: n_blk n_part per kv head (none in a chain)
    int own_blk;               // the own keys' jobs (or the chains): own_blk own_pieces per (kv head, sequence),
    int own_pieces, own_chunk;   // each over own_chunk keys (the last to the end)
    bool own_decode;           // one token: the own keys' jobs are the decode kernel's splits (dec)
    DecodeArgs dec;
    int slots;                 // partials per row: n_part, and own_pieces if own_blk
    float inv_sqrt_hd, softcap;
    float *part, *out;
};

constexpr int kCols = kPrefillNW * kColsPerWave;

// LDS of one workgroup: the columns' rotated q, then the window tiles, then the outputs of all columns;
// or a decode split's.
template <int HD, int NW>
struct DecodeLds {
    DecodeSplitSmem<HD, NW> sm;
    __align__(16) float kd[HD], vd[HD];
    float xnew[8];
};
template <int HD>
constexpr size_t shared_lds() {
    return std::max(std::max(sizeof(PrefillLds<HD>), (size_t)kCols * (HD + 4) * sizeof(float)),
                    sizeof(DecodeLds<HD, kPrefillNW>));
}

// One job: 128 columns (token, head) of one kv head against a range of keys, in the window walk of
// chunked prefill.
template <int HD, bool SOFTCAP, bool NORM, bool PAD>
__global__ __launch_bounds__(64 * kPrefillNW, HD > 128 ? 1 : 2) void shared_kernel(SharedArgs a) {
    constexpr int NW = kPrefillNW;
    constexpr int NKS = HD / 16, NDB = HD / 32, NG = NKS / 4, ROWB = HD / 2;
    const float *const QN = NORM ? a.own.qn : nullptr;
    const int H = a.own.H, G = a.G, T = a.n_tok, hdr = PAD ? a.own.hdr : HD;
    // Jobs of one kv head go to one XCD where the heads divide the XCDs: its streams share an L2.
    const int h = blockIdx.x % H;
    int job = blockIdx.x / H;
    const bool over_prefix = job < a.n_blk * a.n_part;
    // columns: rows (token of a sequence) from row_base on, G heads each; keys: n_pre windows of the
    // prefix from k_begin to k_end, then n_own windows of sequence s_own's own
    int row_base, n_cols, blk, slot, k_begin, k_end, s_own = 0, n_own = 0, own_w0 = 0;
    extern __shared__ __align__(16) unsigned char sh_smem[];
    if (!over_prefix && a.own_decode) {
        job -= a.n_blk * a.n_part;
        const int split = job % a.dec.n_split, gi = job / a.dec.n_split % a.dec.NG;
        DecodeLds<HD, NW> &lds = *reinterpret_cast<DecodeLds<HD, NW> *>(sh_smem);
        decode_split<HD, SOFTCAP, NORM, PAD, NW>(a.dec, split, h * a.dec.NG + gi, job / a.dec.n_split / a.dec.NG, lds.sm,
                                                       lds.kd, lds.vd, lds.xnew);
        return;
    }
    if (over_prefix) {
        blk = job / a.n_part;
        slot = job % a.n_part;
        row_base = 0;
        n_cols = a.own.S * T * G;
        k_begin = slot * a.chunk;
        k_end = min(k_begin + a.chunk, a.prefix_len);
    } else {
        job -= a.n_blk * a.n_part;
        const int piece = job % a.own_pieces;
        job /= a.own_pieces;
        s_own = job / a.own_blk;
        blk = a.own_blk - 1 - job % a.own_blk;  // later tokens first
        slot = a.n_part + piece;
        row_base = s_own * T;
        n_cols = T * G;
        k_begin = 0;
        k_end = a.chain ? a.prefix_len : 0;
        n_own = (min(a.len[s_own] + (min((blk + 1) * kCols, n_cols) - 1) / G + 1, a.own.P) + kWin - 1) / kWin;
        own_w0 = piece * (a.own_chunk / kWin);
        n_own = min(n_own - own_w0, piece + 1 < a.own_pieces ? a.own_chunk / kWin : n_own);
        if (n_own <= 0) {  // (a shorter sequence than the longest: nothing here for the join)
            const int cg = blk * kCols + threadIdx.x;
            if (threadIdx.x < kCols && cg < n_cols) {
                const size_t rows = (size_t)a.own.S * T * a.n_head;
                const size_t r = ((size_t)(row_base + cg / G) * a.n_head + h * G + cg % G) * a.slots + slot;
                a.part[rows * a.slots * HD + r] = kMinit;
                a.part[rows * a.slots * (HD + 1) + r] = 0.0f;
            }
            return;
        }
    }
    const int n_pre = (k_end - k_begin + kWin - 1) / kWin, n_win = n_pre + n_own;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    PrefillLds<HD> &sm = *reinterpret_cast<PrefillLds<HD> *>(sh_smem);
    __shared__ float sm_back[kCols];
    __shared__ int sm_pos[kCols];

    const float qmul = SOFTCAP ? a.inv_sqrt_hd : a.inv_sqrt_hd * kLog2e;
    const int krow = qk_row_key(j);

    const int c_blk = blk * kCols, c_wave = c_blk + wave * kColsPerWave, c = c_wave + j;
    const bool live = c < n_cols;
    const int cc = live ? c : n_cols - 1;
    const int row = row_base + cc / G, s = row / T, tok = row - s * T;
    const int head = h * G + cc % G;

    Pending<HD, NW> pd;
    const DeqConstV dk;
    auto stream_of = [&](const KvLayerView &L, int seq) { return (size_t)seq * H + h; };
    auto fetch = [&](int w) __attribute__((always_inline)) {
        const KvLayerView &L = w < n_pre ? a.pre : a.own;
        const size_t st = stream_of(L, w < n_pre ? a.prefix_seq : s_own);
        fetch_window<HD, NW>(pd, L.kp + st * L.P * ROWB, L.vp + st * (L.P / 32) * (HD * 16), L.ks + st * L.P, L.vs + st * L.P,
                             w < n_pre ? k_begin + w * kWin : (own_w0 + w - n_pre) * kWin, tid, wave);
    };
    fetch(0);

    // q of all columns: read along their rows (a lane that reads its own column's row alone touches a
    // line per 16 bytes: 6 us of a 25 us launch), normalized and rotated, and through LDS to the lanes
    // that multiply it.
    float *const qs = reinterpret_cast<float *>(sh_smem);
    constexpr int V4 = HD / 4, QST = HD + 4, NT = 64 * NW, NQ = kCols * V4 / NT;
    constexpr int QU = NQ < 16 ? NQ : 16;  // (this many rows' loads together)
    float4 x[QU];
    auto load_q = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < QU; u++) {
            const int at = threadIdx.x + NT * (i0 + u), cl = at / V4, d = 4 * (at % V4);
            const int cg = c_blk + cl, ce = min(cg, n_cols - 1), rw = row_base + ce / G;
            const float4 v = *reinterpret_cast<const float4 *>(a.q + ((size_t)rw * a.n_head + h * G + ce % G) * hdr + (d < hdr ? d : 0));
            x[u] = keep4(cg < n_cols && d < hdr, v);
        }
    };
    load_q(0);
    asm volatile("" ::: "memory");  // (on their way before the lengths are waited for)
    const int qslot = a.len[s] + tok;  // the token's own slot
    if (hf == 0) sm_pos[32 * wave + j] = min(rot_of(a.own, s, qslot), a.rope_rows - 1);
    // (min: a graph replayed past the table)
    __syncthreads();
#pragma unroll 1
    for (int i0 = 0; i0 < NQ; i0 += QU) {
        if (i0 > 0) load_q(i0);
        float2 c0[QU], c1[QU];
#pragma unroll
        for (int u = 0; u < QU; u++) {
            const int at = threadIdx.x + NT * (i0 + u), cl = at / V4, d = 4 * (at % V4);
            const int pr = min(d / 2, a.rope_pairs - 1), p1 = min(d / 2 + 1, a.rope_pairs - 1);
            const float *rot = a.rope + (size_t)sm_pos[cl] * a.rope_pairs * 2;
            c0[u] = *reinterpret_cast<const float2 *>(rot + 2 * pr);
            c1[u] = *reinterpret_cast<const float2 *>(rot + 2 * p1);
        }
#pragma unroll
        for (int u = 0; u < QU; u++) {
            const int at = threadIdx.x + NT * (i0 + u), cl = at / V4, d = 4 * (at % V4);
            float4 v = x[u];
            if (QN) {
                float ss = v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
#pragma unroll
                for (int o = 1; o < V4; o <<= 1) ss += __shfl_xor(ss, o, 64);  // (a row's lanes: V4 in a row)
                const float ns = qk_norm_scale_from_sum(ss, hdr, a.own.norm_eps);
                const float4 w = *reinterpret_cast<const float4 *>(QN + (d < hdr ? d : 0));
                v = make_float4(qk_norm_apply(v.x, ns, w.x), qk_norm_apply(v.y, ns, w.y), qk_norm_apply(v.z, ns, w.z),
                                qk_norm_apply(v.w, ns, w.w));
            }
            if (d / 2 < a.rope_pairs) rope_rotate(v.x, v.y, c0[u]);
            if (d / 2 + 1 < a.rope_pairs) rope_rotate(v.z, v.w, c1[u]);
            *reinterpret_cast<float4 *>(qs + cl * QST + d) = v;
        }
    }
    __syncthreads();
    // A power-of-two scale of each column for the hi / lo split, taken back from its scores: a column is
    // another sequence's, whose large, infinite or NaN q must not cost this one its bits.  (Through LDS:
    // in a register it costs the walk spills.)
    const float *const qrow = qs + (32 * wave + j) * QST;
    float mc = 0.0f;
#pragma unroll
    for (int t = 0; t < HD / 8; t++) {
        const floatx4 x = *reinterpret_cast<const floatx4 *>(qrow + 4 * (2 * t + hf));
        mc = fmaxf(fmaxf(mc, fmaxf(fabsf(x[0]), fabsf(x[1]))), fmaxf(fabsf(x[2]), fabsf(x[3])));
    }
    float q_s, q_back;
    q_scale(half_max(mc) * qmul, q_s, q_back);
    sm_back[32 * wave + j] = q_back;
    // the split of this lane's column
    half8 qh[NKS];
    int6v ql1[NG], ql2[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        float lo[32];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int t = 4 * g + u;
            const float *src = qrow + 8 * (2 * t + hf);
            const floatx4 x0 = *reinterpret_cast<const floatx4 *>(src), x1 = *reinterpret_cast<const floatx4 *>(src + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = opaque((kPerm[e] < 4 ? x0[kPerm[e] & 3] : x1[kPerm[e] & 3]) * (qmul * q_s));
                const _Float16 hi = (_Float16)v;
                qh[t][e] = hi;
                lo[8 * u + e] = v - (float)hi;
            }
        }
        q_lo_terms(lo, ql1[g], ql2[g]);
    }
    __syncthreads();  // (the windows' tiles take q's place)

    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) o[db] = (floatx16)0.0f;
    float m_run = 0.0f, l_run = 0.0f;
    bool first = true;

    stage_codes<HD, NW>(sm, 0, pd, tid, wave, dk);
    stage_scales<HD, NW, true>(sm, 0, pd, tid, 1.0f);
    if (1 < n_win) fetch(1);
    __syncthreads();

    for (int w = 0; w < n_win; w++) {
        const int buf = w & 1;
        floatx16 sc[2] = {(floatx16)0.0f, (floatx16)0.0f};
        __builtin_amdgcn_s_setprio(3);
        using PD = Pending<HD, NW>;
        constexpr int NPART = PD::SPLIT ? 0 : 8 * PD::NK;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            half8 ka0[4], ka1[4];
            ka0[0] = sm.k[buf][krow][k_slot<HD>(krow, 2 * (4 * g) + hf)];
            ka1[0] = sm.k[buf][32 + krow][k_slot<HD>(32 + krow, 2 * (4 * g) + hf)];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int t = 4 * g + u;
                if (u + 1 < 4) {
                    ka0[u + 1] = sm.k[buf][krow][k_slot<HD>(krow, 2 * (t + 1) + hf)];
                    ka1[u + 1] = sm.k[buf][32 + krow][k_slot<HD>(32 + krow, 2 * (t + 1) + hf)];
                }
                __builtin_amdgcn_sched_barrier(0);
                sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka0[u], qh[t], sc[0], 0, 0, 0);
                sc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka1[u], qh[t], sc[1], 0, 0, 0);
                if constexpr (NPART > 0) {
#pragma unroll
                    for (int part = t * NPART / NKS; part < (t + 1) * NPART / NKS; part++)
                        stage_part<HD, NW>(sm, buf ^ 1, pd, tid, part, dk);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            const int6v k0 = fp6_of(ka0, 1.0f), k1 = fp6_of(ka1, 1.0f);
            sc[0] = mfma_lo6(k0, ql1[g], sc[0], kQlo1E8);
            sc[1] = mfma_lo6(k1, ql1[g], sc[1], kQlo1E8);
            sc[0] = mfma_lo6(k0, ql2[g], sc[0], kQlo2E8);
            sc[1] = mfma_lo6(k1, ql2[g], sc[1], kQlo2E8);
        }
        if constexpr (NPART == 0) stage_codes<HD, NW>(sm, buf ^ 1, pd, tid, wave, dk);
        __builtin_amdgcn_s_setprio(0);
        if (w + 1 < n_win) stage_scales<HD, NW, true>(sm, buf ^ 1, pd, tid, 1.0f);
        if (w + 2 < n_win) fetch(w + 2);
        // Keys are numbered within their stream: a column sees the prefix up to k_end, its own keys up to
        // its slot.
        const bool pre = w < n_pre;
        const int base = pre ? k_begin + w * kWin : (own_w0 + w - n_pre) * kWin;
        const int qpos = !live ? -1 : pre ? k_end - 1 : qslot;
        const int len_w = pre ? 0 : a.len[s_own];
        const int qmin_w = pre ? k_end - 1 : len_w + c_wave / G;
        const int qmax_w = pre ? k_end - 1 : len_w + (min(c_wave + kColsPerWave, n_cols) - 1) / G;
        if (c_wave < n_cols && base <= qmax_w) {
            const float q_back = sm_back[32 * wave + j];
            sc[0] *= q_back;
            sc[1] *= q_back;
            const bool mask = base + kWin - 1 > qmin_w;
            window_scores<NDB, SOFTCAP>(sc, sm.sk[buf], sm.svlog[buf], a.softcap, mask, first, base, hf, qpos, m_run,
                                        l_run, o);
            first = false;
#pragma unroll
            for (int st = 0; st < 4; st++) {
                half8 pb, pl;
                step_probs<true>(sc, sm.sv[buf], st, hf, l_run, pb, pl);
                __builtin_amdgcn_s_setprio(2);
                half8 va[NDB];
#pragma unroll
                for (int db = 0; db < NDB; db++) {
                    const int vr = 32 * db + j;
                    va[db] = sm.v[buf][vr][v_slot(vr, 2 * st + hf)];
                }
#pragma unroll
                for (int db = 0; db < NDB; db++) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[db], pb, o[db], 0, 0, 0);
#pragma unroll
                for (int db = 0; db < NDB; db++) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[db], pl, o[db], 0, 0, 0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    }

    const float l = half_sum(l_run);
    const size_t rows = (size_t)a.own.S * T * a.n_head;
    const size_t row_head = (size_t)row * a.n_head + head;
    // The outputs go through LDS (the windows' place), whole rows from there.
    constexpr int OST = HD + 4;
    float *const mo = reinterpret_cast<float *>(sh_smem);
    const float e0 = !a.chain ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int q = 0; q < 4; q++)
            *reinterpret_cast<floatx4 *>(mo + (32 * wave + j) * OST + 32 * db + 8 * q + 4 * hf) =
                e0 * (floatx4){o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]};
    if (!a.chain && live && hf == 0) {
        a.part[rows * a.slots * HD + row_head * a.slots + slot] = first ? kMinit : m_run;  // (a wave without a window)
        a.part[rows * a.slots * (HD + 1) + row_head * a.slots + slot] = l;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < kCols * V4; x += NT) {
        const int cl = x / V4, d = 4 * (x % V4), cg = c_blk + cl;
        if (cg >= n_cols) break;
        const size_t rh = (size_t)(row_base + cg / G) * a.n_head + h * G + cg % G;
        float *dst = a.chain ? a.out + rh * hdr : a.part + (rh * a.slots + slot) * HD;
        if (d < hdr) *reinterpret_cast<floatx4 *>(dst + d) = *reinterpret_cast<floatx4 *>(mo + cl * OST + d);
    }
}

struct JoinArgs {
    const float *part;  // [rows][slots][HD], m, l
    const float *own;   // the decode kernel's partials, or null
    const int32_t *len;
    float *out;
    int rows, slots, n_head, H, n_tok, hdr;
    int own_split, own_chunk, hlen, cap;  // of the decode plan; cap: positions of the own cache
};

// The join of one (token, head) row's parts by NWR waves: lane l holds HD / 64 dims, wave w every NWR-th
// group of 8 parts, whose loads do not depend on each other.
template <int HD, int NWR>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
    constexpr int D = HD / 64, RPW = 4 / NWR;  // rows per workgroup
    __shared__ float acc_s[4][HD], l_s[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wr = wave % NWR;
    // (rows of one kv head on the XCD that wrote their parts)
    const int u = blockIdx.x / a.H * RPW + wave / NWR, G = a.n_head / a.H;
    const bool some = u < a.rows / a.H;
    const int uc = some ? u : a.rows / a.H - 1;
    const int tok = uc / G, s = tok / a.n_tok;
    const int row = tok * a.n_head + blockIdx.x % a.H * G + uc % G, r = row;
    const int qpos = (a.hlen >= 0 ? a.hlen : a.len[s]) + tok - s * a.n_tok;
    const float *po = a.part + (size_t)r * a.slots * HD, *pm = a.part + (size_t)a.rows * a.slots * HD + (size_t)r * a.slots;
    const float *pl = pm + (size_t)a.rows * a.slots;
    // (a graph replayed past the cache's capacity: the own part was not written, nor is the output)
    const bool ok = some && qpos < a.cap;
    const int n_own = a.own && ok ? min((qpos + a.own_chunk) / a.own_chunk, a.own_split) : 0;
    const float *oo = nullptr, *om = nullptr, *ol = nullptr;
    if (a.own) {
        oo = a.own + (size_t)r * a.own_split * HD;
        om = a.own + (size_t)a.rows * a.own_split * HD + (size_t)r * a.own_split;
        ol = om + (size_t)a.rows * a.own_split;
    }
    const int n = a.slots + n_own;
    float M = kMinit;
    for (int i = lane; i < n; i += 64) M = fmaxf(M, i < a.slots ? pm[i] : om[i - a.slots]);
    M = wave_max(M);
    float acc[D] = {}, l = 0.0f;
    for (int i0 = 8 * wr; i0 < n; i0 += 8 * NWR) {
        float x[8][D], w[8], ls[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = min(i0 + k, n - 1);
            const bool pre = i < a.slots;
            const float *src = pre ? po + (size_t)i * HD : oo + (size_t)(i - a.slots) * HD;
#pragma unroll
            for (int e = 0; e < D; e++) x[k][e] = src[D * lane + e];
            w[k] = pre ? pm[i] : om[i - a.slots];
            ls[k] = pre ? pl[i] : ol[i - a.slots];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i0 + k >= n) break;
            const float e2 = __builtin_amdgcn_exp2f(w[k] - M);
            if (ls[k] == 0.0f) continue;  // (a part without keys has no output; one of a NaN q has)
#pragma unroll
            for (int e = 0; e < D; e++) acc[e] += e2 * x[k][e];
            l += e2 * ls[k];
        }
    }
    if constexpr (NWR > 1) {
#pragma unroll
        for (int e = 0; e < D; e++) acc_s[wave][D * lane + e] = acc[e];
        if (lane == 0) l_s[wave] = l;
        __syncthreads();
        if (wr != 0) return;
#pragma unroll
        for (int k = 1; k < NWR; k++) {
#pragma unroll
            for (int e = 0; e < D; e++) acc[e] += acc_s[wave + k][D * lane + e];
            l += l_s[wave + k];
        }
    }
    if (!ok) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float *o = a.out + (size_t)row * a.hdr;
#pragma unroll
    for (int e = 0; e < D; e++)
        if (D * lane + e < a.hdr) o[D * lane + e] = acc[e] * inv;
}

}  // namespace

// A chain needs no partials and no join, but its columns are one sequence's: taken for chunks that fill
// blocks of 128 to 3/4 and more than half of the chip with blocks.  32 heads over 8 of 128 dims, 4097 shared
// keys, with and without: 8 x 256 tokens 254 and 308 us, 8 x 96 164 and 183, 4 x 130 165 and 175, 32 x 24
// (3/4 filled) 160 and 184; below: 32 x 16 (half filled) 159 and 107, 8 x 64 (half of the chip) 163 and
// 108, 2 x 256 170 and 110.
static bool chains(int n_seq, int n_tok, int G, int n_kv, int n_cu) {
    const int64_t cols = (int64_t)n_tok * G, blk = (cols + kCols - 1) / kCols;
    return n_tok > 1 && 4 * cols >= 3 * blk * kCols && 2 * blk * n_seq * n_kv > n_cu;
}

// Pieces of own keys for a chunk that is no chain: until the jobs fill the chip, of 256 keys at least.  4 x 3
// tokens over 2000 own keys 27 us, in one piece 63; 8 x 16 over 1000 49 us, until half of the chip 51, in
// one piece 69.
static int own_pieces(int n_seq, int own_blk, int n_kv, int own_max, int n_cu) {
    const int64_t jobs = (int64_t)n_seq * own_blk * n_kv;
    return (int)std::max<int64_t>(1, std::min<int64_t>(n_cu / jobs, (own_max + 255) / 256));
}

SharedPlan shared_plan(int n_seq, int n_tok, int G, int n_kv, int prefix_len, int own_max, int n_cu) {
    SharedPlan p;
    p.chain = chains(n_seq, n_tok, G, n_kv, n_cu);
    p.n_blk = p.n_part = p.chunk = 0;
    p.own_blk = n_tok > 1 ? (n_tok * G + kCols - 1) / kCols : 0;
    p.own_pieces = 1;
    p.own_chunk = 0;
    if (p.chain) return p;
    if (p.own_blk) {
        const int n = own_pieces(n_seq, p.own_blk, n_kv, own_max, n_cu);
        p.own_chunk = ((own_max + n - 1) / n + kWin - 1) / kWin * kWin;
        p.own_pieces = (own_max + p.own_chunk - 1) / p.own_chunk;
    }
    // Pieces of the prefix: one job per CU, and a window at least in each.  (Two groups of waves in a workgroup,
    // each with every second window, were slower from 1000 shared keys on: 8 x 16 tokens 48 us, 42 with one
    // group and a piece per CU.)
    p.n_blk = (int)(((int64_t)n_seq * n_tok * G + kCols - 1) / kCols);
    const int64_t streams = (int64_t)p.n_blk * n_kv;
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>(n_cu / streams, (prefix_len + kWin - 1) / kWin));
    p.chunk = (int)((prefix_len + n - 1) / n + kWin - 1) / kWin * kWin;
    p.n_part = (prefix_len + p.chunk - 1) / p.chunk;
    return p;
}

// One token: the own keys in splits of at least 512 (two rounds of a workgroup's windows), longer ones where
// the batch has more than fill the chip.  One sequence of 16000 17.2 us, with 1024 20.5; two of 4000 15.3 and
// 16.2; 16 of 700 to 1500 30.2 and 27.6.  With 256: 32 of 60 to 500 31.2 us, 30.2 with 512, else the same.
void shared_own_plan(const int32_t *n_ctx, int n_seq, int n_kv, int G, int n_cu, int *chunk, int *n_split) {
    constexpr int64_t kMinSplit = 512;
    int64_t total = 0;
    int most = 1;
    for (int s = 0; s < n_seq; s++) {
        total += n_ctx[s];
        most = std::max(most, (int)n_ctx[s]);
    }
    const int64_t per_cu = (total * n_kv * ((G + 7) / 8) + n_cu - 1) / n_cu;
    *chunk = (int)(std::max(kMinSplit, per_cu) + 63) / 64 * 64;
    *n_split = (most + *chunk - 1) / *chunk;
}

int shared_slots_cap(int n_seq, int n_tok, int G, int n_kv, int max_prefix, int own_max, int n_cu) {
    if (chains(n_seq, n_tok, G, n_kv, n_cu)) return 0;
    const int64_t streams = ((int64_t)n_seq * n_tok * G + kCols - 1) / kCols * n_kv;
    const int pre = (int)std::max<int64_t>(1, std::min<int64_t>(n_cu / streams, (max_prefix + kWin - 1) / kWin));
    return pre + (n_tok > 1 ? own_pieces(n_seq, (n_tok * G + kCols - 1) / kCols, n_kv, own_max, n_cu) : 0);
}

hipError_t launch_shared(const SharedCall &c, hipStream_t st) {
    SharedArgs a;
    a.own = c.own;
    a.pre = c.pre;
    a.prefix_seq = c.prefix_seq;
    a.prefix_len = c.prefix_len;
    a.len = c.d_len;
    a.q = c.q;
    a.rope = c.rope;
    a.rope_pairs = c.rope_pairs;
    a.rope_rows = c.rope_rows;
    a.n_head = c.n_head;
    a.G = c.n_head / c.own.H;
    a.n_tok = c.n_tok;
    a.chain = c.plan.chain;
    a.n_blk = c.plan.n_blk;
    a.n_part = c.plan.n_part;
    a.chunk = c.plan.chunk;
    a.own_blk = c.plan.own_blk;
    a.own_decode = c.own_part != nullptr;
    a.own_pieces = c.plan.own_pieces;
    a.own_chunk = c.plan.own_chunk;
    a.slots = a.n_part + (a.own_blk ? a.own_pieces : 0);
    a.inv_sqrt_hd = 1.0f / sqrtf((float)c.own.hdr);
    a.softcap = c.softcap;
    a.part = c.part;
    a.out = c.out;
    int own_jobs = a.own_blk * a.own_pieces * c.own.S;  // per kv head
    if (c.own_part) {
        DecodeArgs &d = a.dec;
        d = {};
        d.L = c.own;
        d.len = c.d_len;
        d.hlen = c.hlen;
        d.q = c.q;
        d.rope = c.rope;
        d.rope_pairs = c.rope_pairs;
        d.n_head = c.n_head;
        d.Gt = a.G;
        d.NG = (a.G + 7) / 8;
        d.G = std::min(a.G, 8);
        d.chunk = c.own_chunk;
        d.n_split = c.own_split;
        d.inv_sqrt_hd = a.inv_sqrt_hd;
        d.softcap = c.softcap;
        d.out = c.out;
        d.ws = c.own_part;
        d.k_new = c.k_new;
        d.v_new = c.v_new;
        own_jobs = d.n_split * d.NG * c.own.S;
    }
    const unsigned jobs = (unsigned)((a.n_blk * a.n_part + own_jobs) * c.own.H);
    const bool cap = c.softcap > 0.0f, norm = c.own.qn != nullptr || c.own.kn != nullptr;
#define TS_SH3(HDV, SC, NM, PD)                                                                      \
    {                                                                                                \
        constexpr size_t lds = shared_lds<HDV>();                                                    \
        static_assert(lds <= 156 * 1024, "a workgroup's windows fit a CU's LDS");                     \
        if (lds > 64 * 1024)                                                                         \
            (void)hipFuncSetAttribute((const void *)shared_kernel<HDV, SC, NM, PD>,                  \
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);         \
        shared_kernel<HDV, SC, NM, PD><<<jobs, 64 * kPrefillNW, lds, st>>>(a);                       \
    }
#define TS_SH2(HDV, PD)                                                                              \
    {                                                                                                \
        if (cap) { if (norm) TS_SH3(HDV, true, true, PD) else TS_SH3(HDV, true, false, PD) }         \
        else { if (norm) TS_SH3(HDV, false, true, PD) else TS_SH3(HDV, false, false, PD) }           \
    }
#define TS_SH(HDV) { if (c.own.hdr != c.own.hd) TS_SH2(HDV, true) else TS_SH2(HDV, false) }
    if (c.own.hd == 256) TS_SH(256)
    else if (c.own.hd == 128) TS_SH(128)
    else TS_SH(64)
#undef TS_SH
#undef TS_SH2
#undef TS_SH3
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.chain) return e;
    JoinArgs ja;
    ja.part = c.part;
    ja.own = c.own_part;
    ja.len = c.d_len;
    ja.out = c.out;
    ja.rows = c.own.S * c.n_tok * c.n_head;
    ja.slots = a.slots;
    ja.n_head = c.n_head;
    ja.H = c.own.H;
    ja.n_tok = c.n_tok;
    ja.hdr = c.own.hdr;
    ja.own_split = c.own_split;
    ja.own_chunk = c.own_chunk;
    ja.hlen = c.hlen;
    ja.cap = c.own.P;
    // Few rows: all four waves of a workgroup on one row's parts, where a wave to a row leaves CUs idle.  One
    // token of 32 heads, with and without: 4 sequences 23.1 and 26.0 us, 32 30.5 and 31.5, 64 42.1 and 41.0, 128
    // 66.4 and 63.1.
    const bool wide = ja.rows <= 4 * c.n_cu;
    const unsigned blocks = wide ? ja.rows : (ja.rows / ja.H + 3) / 4 * ja.H;
#define TS_JOIN(HDV) \
    { if (wide) join_kernel<HDV, 4><<<blocks, 256, 0, st>>>(ja); else join_kernel<HDV, 1><<<blocks, 256, 0, st>>>(ja); }
    if (c.own.hd == 256) TS_JOIN(256)
    else if (c.own.hd == 128) TS_JOIN(128)
    else TS_JOIN(64)
#undef TS_JOIN
    return hipGetLastError();
}

}  // namespace ts
