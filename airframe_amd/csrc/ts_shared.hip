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
#include "ts_shared.h"

#include "ts_window.h"

namespace ts {
namespace {

struct SharedArgs {
    KvLayerView own, pre;
    int prefix_seq, prefix_len;
    const int32_t *len;
    const float *q, *rope;
    int rope_pairs, rope_rows, n_head, G, n_tok;
    int n_blk, n_part, chunk;  // the prefix's jobs: n_blk n_part per kv head
    int own_blk;               // the own keys' jobs: own_blk per (kv head, sequence); 0 without
    int slots;                 // partials per row: n_part, and one of the own keys if own_blk
    float inv_sqrt_hd, softcap;
    float *part;
};

// One job: 128 columns (token, head) of one kv head against a range of one stream's keys, in the
// window walk of chunked prefill.
template <int HD, bool SOFTCAP, bool NORM, bool PAD>
__global__ __launch_bounds__(64 * kPrefillNW, HD > 128 ? 1 : 2) void shared_kernel(SharedArgs a) {
    constexpr int NW = kPrefillNW;
    constexpr int NKS = HD / 16, NDB = HD / 32, NG = NKS / 4, ROWB = HD / 2;
    constexpr int COLS = NW * kColsPerWave;
    const float *const QN = NORM ? a.own.qn : nullptr;
    const int H = a.own.H, G = a.G, T = a.n_tok, hdr = PAD ? a.own.hdr : HD;
    // Jobs of one kv head go to one XCD where the heads divide the XCDs: its streams share an L2.
    const int h = blockIdx.x % H;
    int job = blockIdx.x / H;
    const bool over_prefix = job < a.n_blk * a.n_part;
    int row_base, n_cols, blk, slot, k_begin, k_end, s_str;
    const KvLayerView &L = over_prefix ? a.pre : a.own;
    if (over_prefix) {
        blk = job / a.n_part;
        slot = job % a.n_part;
        row_base = 0;
        n_cols = a.own.S * T * G;
        s_str = a.prefix_seq;
        k_begin = slot * a.chunk;
        k_end = min(k_begin + a.chunk, a.prefix_len);
    } else {
        job -= a.n_blk * a.n_part;
        s_str = job / a.own_blk;
        blk = a.own_blk - 1 - job % a.own_blk;  // later tokens first
        slot = a.n_part;
        row_base = s_str * T;
        n_cols = T * G;
        k_begin = 0;
        k_end = min(a.len[s_str] + (min((blk + 1) * COLS, n_cols) - 1) / G + 1, L.P);
    }
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    extern __shared__ __align__(16) unsigned char sh_smem[];
    PrefillLds<HD> &sm = *reinterpret_cast<PrefillLds<HD> *>(sh_smem);
    __shared__ float sm_qb[NW];

    const size_t stream = (size_t)s_str * H + h;
    const uint8_t *kbase = L.kp + stream * L.P * ROWB;
    const uint8_t *vbase = L.vp + stream * (L.P / 32) * (HD * 16);
    const float *ksb = L.ks + stream * L.P, *vsb = L.vs + stream * L.P;
    const float qmul = SOFTCAP ? a.inv_sqrt_hd : a.inv_sqrt_hd * kLog2e;
    const int krow = qk_row_key(j);

    const int c_blk = blk * COLS, c_wave = c_blk + wave * kColsPerWave, c = c_wave + j;
    const bool live = c < n_cols;
    const int cc = live ? c : n_cols - 1;
    const int row = row_base + cc / G, s = row / T, tok = row - s * T;
    const int head = h * G + cc % G;
    const float *qrow = a.q + ((size_t)row * a.n_head + head) * hdr;
    const int len_s = a.len[s];
    const int qslot = len_s + tok;  // the token's own slot
    // the last key this column sees
    const int qpos = !live ? -1 : over_prefix ? k_end - 1 : qslot;
    const int len0 = over_prefix ? 0 : len_s;  // (one sequence per own job)
    const int qmin_w = over_prefix ? k_end - 1 : len0 + c_wave / G;
    const int qmax_w = c_wave >= n_cols ? -1
                       : over_prefix    ? k_end - 1
                                        : len0 + (min(c_wave + kColsPerWave, n_cols) - 1) / G;

    Pending<HD, NW> pd;
    const DeqConstV dk;
    fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, k_begin, tid, wave);

    // q of this lane's column: norm, rotation at its position, power-of-two scale, hi/lo split
    const float ns = QN ? qk_norm_scale(qrow, hdr, a.own.norm_eps) : 1.0f;
    float q_s, inv_s;
    half8 qh[NKS];
    int6v ql1[NG], ql2[NG];
    {
        float xq[NKS][8];
        float2 cs[NKS][4];
        const int qrot = min(rot_of(a.own, s, qslot), a.rope_rows - 1);  // (a graph replayed past the table)
        float qb = 0.0f;
#pragma unroll
        for (int t = 0; t < NKS; t++) {
            q_read8(qrow, 2 * t + hf, QN, ns, xq[t], hdr);
            load_rot8(a.rope, a.rope_pairs, 2 * t + hf, qrot, cs[t]);
            qb = fmaxf(qb, fmaxf(fmaxf(fabsf(xq[t][0]) + fabsf(xq[t][1]), fabsf(xq[t][2]) + fabsf(xq[t][3])),
                                 fmaxf(fabsf(xq[t][4]) + fabsf(xq[t][5]), fabsf(xq[t][6]) + fabsf(xq[t][7]))));
        }
        qb = wave_max(qb);
        if (lane == 0) sm_qb[wave] = qb;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) qb = fmaxf(qb, sm_qb[w]);
        q_scale(qb * qmul, q_s, inv_s);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float lo[32];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int t = 4 * g + u;
                split_q8_f32(xq[t], cs[t], 2 * t + hf, a.rope_pairs, qmul * q_s, qh[t], lo + 8 * u);
                if (!live) {
                    qh[t] = (half8)(_Float16)0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) lo[8 * u + e] = 0.0f;
                }
            }
            q_lo_terms(lo, ql1[g], ql2[g]);
        }
    }

    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) o[db] = (floatx16)0.0f;
    float m_run = 0.0f, l_run = 0.0f;
    bool first = true;
    const int n_win = (k_end - k_begin + kWin - 1) / kWin;

    stage_codes<HD, NW>(sm, 0, pd, tid, wave, dk);
    stage_scales<HD, NW, true>(sm, 0, pd, tid, inv_s);
    if (n_win > 1) fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, k_begin + kWin, tid, wave);
    __syncthreads();

    for (int w = 0; w < n_win; w++) {
        const int buf = w & 1, base = k_begin + w * kWin;
        const bool more = w + 1 < n_win;
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
        if (more) stage_scales<HD, NW, true>(sm, buf ^ 1, pd, tid, inv_s);
        if (w + 2 < n_win) fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, base + 2 * kWin, tid, wave);
        if (base <= qmax_w) {
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
    if (live) {
        const size_t rows = (size_t)a.own.S * T * a.n_head;
        const size_t r = ((size_t)row * a.n_head + head) * a.slots + slot;
        float *dst = a.part + r * HD;
#pragma unroll
        for (int db = 0; db < NDB; db++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (32 * db + 8 * q + 4 * hf < hdr)
                    *reinterpret_cast<float4 *>(dst + 32 * db + 8 * q + 4 * hf) =
                        make_float4(o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]);
        if (hf == 0) {
            a.part[rows * a.slots * HD + r] = m_run;
            a.part[rows * a.slots * (HD + 1) + r] = l;
        }
    }
}

struct JoinArgs {
    const float *part;  // [rows][slots][HD], m, l
    const float *own;   // the decode kernel's partials, or null
    const int32_t *len;
    float *out;
    int rows, slots, n_head, n_tok, hdr;
    int own_split, own_chunk, hlen, cap;  // of the decode plan; cap: positions of the own cache
};

// The join of one (token, head) row's parts, one wave each: lane l holds HD / 64 dims.  The parts'
// loads do not depend on each other (8 at a time), so a row costs about two memory round trips.
template <int HD>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
    constexpr int D = HD / 64;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const int tok = row / a.n_head, s = tok / a.n_tok;
    const int qpos = (a.hlen >= 0 ? a.hlen : a.len[s]) + tok - s * a.n_tok;
    // (a graph replayed past the cache's capacity: the own part was not written, nor is the output)
    if (qpos >= a.cap) return;
    const float *po = a.part + (size_t)row * a.slots * HD, *pm = a.part + (size_t)a.rows * a.slots * HD + (size_t)row * a.slots;
    const float *pl = pm + (size_t)a.rows * a.slots;
    const int n_own = a.own ? min((qpos + a.own_chunk) / a.own_chunk, a.own_split) : 0;
    const float *oo = nullptr, *om = nullptr, *ol = nullptr;
    if (a.own) {
        oo = a.own + (size_t)row * a.own_split * HD;
        om = a.own + (size_t)a.rows * a.own_split * HD + (size_t)row * a.own_split;
        ol = om + (size_t)a.rows * a.own_split;
    }
    const int n = a.slots + n_own;
    float M = kMinit;
    for (int i = lane; i < n; i += 64) M = fmaxf(M, i < a.slots ? pm[i] : om[i - a.slots]);
    M = wave_max(M);
    float acc[D] = {}, l = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 8) {
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
#pragma unroll
            for (int e = 0; e < D; e++) acc[e] += e2 * x[k][e];
            l += e2 * ls[k];
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    float *o = a.out + (size_t)row * a.hdr;
#pragma unroll
    for (int e = 0; e < D; e++)
        if (D * lane + e < a.hdr) o[D * lane + e] = acc[e] * inv;
}

constexpr int kCols = kPrefillNW * kColsPerWave;
constexpr int kMinPart = 256;  // keys of a piece, at least: a piece costs a row of partials per column

}  // namespace

int shared_parts_cap(int n_rows, int G, int n_kv, int max_prefix, int stored_hd, int n_cu) {
    const int64_t streams = ((int64_t)n_rows * G + kCols - 1) / kCols * n_kv;
    const int64_t target = (int64_t)n_cu;
    return (int)std::max<int64_t>(1, std::min<int64_t>(target / streams, (max_prefix + kMinPart - 1) / kMinPart));
}

SharedPlan shared_plan(int n_rows, int G, int n_kv, int prefix_len, int stored_hd, int n_cu) {
    SharedPlan p;
    p.n_blk = (int)(((int64_t)n_rows * G + kCols - 1) / kCols);
    const int n = shared_parts_cap(n_rows, G, n_kv, prefix_len, stored_hd, n_cu);
    p.chunk = ((prefix_len + n - 1) / n + kWin - 1) / kWin * kWin;
    p.n_part = (prefix_len + p.chunk - 1) / p.chunk;
    return p;
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
    a.n_blk = c.plan.n_blk;
    a.n_part = c.plan.n_part;
    a.chunk = c.plan.chunk;
    a.own_blk = c.own_part ? 0 : (c.n_tok * a.G + kCols - 1) / kCols;
    a.slots = a.n_part + (a.own_blk ? 1 : 0);
    a.inv_sqrt_hd = 1.0f / sqrtf((float)c.own.hdr);
    a.softcap = c.softcap;
    a.part = c.part;
    const unsigned jobs = (unsigned)((a.n_blk * a.n_part + a.own_blk * c.own.S) * c.own.H);
    const bool cap = c.softcap > 0.0f, norm = c.own.qn != nullptr;
#define TS_SH3(HDV, SC, NM, PD)                                                                      \
    {                                                                                                \
        constexpr size_t lds = sizeof(PrefillLds<HDV>);                                              \
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
    if (e != hipSuccess) return e;
    JoinArgs ja;
    ja.part = c.part;
    ja.own = c.own_part;
    ja.len = c.d_len;
    ja.out = c.out;
    ja.rows = c.own.S * c.n_tok * c.n_head;
    ja.slots = a.slots;
    ja.n_head = c.n_head;
    ja.n_tok = c.n_tok;
    ja.hdr = c.own.hdr;
    ja.own_split = c.own_plan.n_split;
    ja.own_chunk = c.own_plan.chunk;
    ja.hlen = c.hlen;
    ja.cap = c.own.P;
    const unsigned blocks = (ja.rows + 3) / 4;
    if (c.own.hd == 256) join_kernel<256><<<blocks, 256, 0, st>>>(ja);
    else if (c.own.hd == 128) join_kernel<128><<<blocks, 256, 0, st>>>(ja);
    else join_kernel<64><<<blocks, 256, 0, st>>>(ja);
    return hipGetLastError();
}

}  // namespace ts
