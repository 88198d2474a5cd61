// ts_prefill.hip -- chunked-prefill causal attention over the INT4 cache for gfx950.
//
// Semantics: the CPU reference attention with a KV cache (src/ops/reference/attention.rs:
// 236-313, causal mask softmax.rs:104-109): query t of the chunk sits at absolute position
// len+t and attends to positions 0..len+t of the dequantized INT4 cache.  It replaces the f32
// main_attn_out used by batched prefill (sh_layer_v1.wgsl:662-762), which recomputes every
// score per output element, with matrix-core tiles:
//
// * The (query token, head) pairs that share one kv head form the columns of the MFMA
//   N dimension: column c of a (sequence, kv head) is token c / G, head c % G.
// * grid = (column block of 128, kv head, sequence); each of the 4 waves owns 32 columns,
//   one N tile of v_mfma_f32_32x32x16_f16 (half the instructions of 16x16x32 for the same
//   work).  The workgroup walks the keys in 64-key windows:
//   every thread loads one 16-byte piece of the next window's K rows / V blocks / scales
//   while the current window is computed, then converts it to exact f16 integer codes in a
//   double-buffered LDS tile, so each code is converted once per workgroup and read by all
//   4 waves.
// * S^T = K Q^T with q split into an f16 high half (f16 MFMAs) and a low half as two fp6 terms
//   (one scaled fp6 MFMA per term and 64 dims, the K codes converted to fp6 from the same f16
//   operand registers), all into one f32 accumulator, with 1/sqrt(hd)*log2(e) and a
//   power-of-two range scale folded into q.  K rows enter the MFMA in
//   the order that leaves every lane holding, per 16-key step, exactly the 8 keys it supplies
//   to the PV operand, so P never moves between lanes.  The score is scaled by s_k in f32,
//   masked only in windows that cross the causal diagonal, and enters an online softmax in
//   the exp2 domain whose running max is raised lazily; p*s_v goes to O^T += V^T P^T split
//   hi + lo in f16 (two MFMAs) under an exponent bound that keeps it below 2^15.
// * Each wave owns whole output rows, so the result is written straight from registers.
#include "ts_window.h"

namespace ts {
namespace {

struct PrefillArgs {
    KvLayerView L;
    const int32_t *len;
    const float *q;
    const float *rope;
    int rope_pairs;
    int n_head;
    int G;
    int n_tok;
    float inv_sqrt_hd;
    float softcap;
    float *out;
    int q_delay;  // sleeps of ~1 us before the q read of the lightest column block (0: none)
};

// PAD: the caller's head dim L.hdr is below the stored HD (q and output rows of hdr floats).
template <int HD, bool SOFTCAP, bool NORM, bool PAD>
__global__ __launch_bounds__(64 * kPrefillNW, HD > 128 ? 1 : 2) void prefill_kernel(PrefillArgs a) {
    constexpr int NW = kPrefillNW;
    constexpr int NKS = HD / 16;   // MFMA k-steps over the head dim
    constexpr int NDB = HD / 32;   // 32-dim output tiles
    constexpr int NG = NKS / 4;    // groups of 4 k-steps (one fp6 MFMA each)
    constexpr int ROWB = HD / 2;
    constexpr int COLS = NW * kColsPerWave;  // columns per block
    const KvLayerView &L = a.L;
    const float *const QN = NORM ? L.qn : nullptr;  // QK norm of q (compiled out when off)
    // Workgroups are dispatched round robin over the 8 XCDs by linear id.  Give XCD x the
    // contiguous range [x*N/8, (x+1)*N/8) of (column block, kv head, sequence) in row order, so
    // the 16-odd blocks that read one (sequence, kv head) stream share an L2 and every XCD gets
    // the same mix of long and short blocks.
    int xb = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    {
        const int n_wg = gridDim.x * gridDim.y * gridDim.z;
        if (n_wg % 8 == 0) {
            const int id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
            // Two workgroups share a CU.  The dispatch order within an XCD is reversed in
            // every second round of 32 (its CU count), so that a CU's two workgroups tend to
            // be one heavy (late-token) and one light block (4% faster on a 4 x 512-token
            // prefill).  The reversal is a permutation of the XCD's range.
            const int per = n_wg / 8;
            int k = id / 8;
            if ((k >> 5) & 1) {
                const int r0 = k & ~31, rl = min(32, per - r0);
                k = r0 + rl - 1 - (k - r0);
            }
            const int logical = (id % 8) * per + k;
            xb = logical % gridDim.x;
            h = (logical / gridDim.x) % gridDim.y;
            s = logical / (gridDim.x * gridDim.y);
        }
    }
    const int G = a.G;
    const int n_cols = a.n_tok * G;
    const int n_blk = (n_cols + COLS - 1) / COLS;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;  // MFMA column / lane half
    const int len0 = a.len[s];
    // (dynamic: the hd-256 tiles take 128 KB)
    extern __shared__ __align__(16) unsigned char pf_smem[];
    PrefillLds<HD> &sm = *reinterpret_cast<PrefillLds<HD> *>(pf_smem);
    __shared__ float sm_qb[NW];

    const size_t row = (size_t)s * L.H + h;
    const uint8_t *kbase = L.kp + row * L.P * ROWB;
    const uint8_t *vbase = L.vp + row * (L.P / 32) * (HD * 16);
    const float *ksb = L.ks + row * L.P;
    const float *vsb = L.vs + row * L.P;
    const float qmul = SOFTCAP ? a.inv_sqrt_hd : a.inv_sqrt_hd * kLog2e;
    const int krow = qk_row_key(j);  // K row this lane feeds to the QK MFMA (within 32 keys)

    // Heavier column blocks (later tokens) first.
    const int cblk = n_blk - 1 - xb;
    const int c_blk = cblk * COLS;
    const int c_wave = c_blk + wave * kColsPerWave;
    const int c = c_wave + j;
    const bool live = c < n_cols;
    const int cc = live ? c : n_cols - 1;
    const int tok = cc / G;
    const int hdr = PAD ? L.hdr : HD;  // row length of q and the output (stored dims past it are 0)
    const float *qrow = a.q + (((size_t)s * a.n_tok + tok) * a.n_head + h * G + cc % G) * hdr;
    const int qpos = live ? len0 + tok : -1;

    // The first window's K and V loads go out before q is read.
    Pending<HD, NW> pd;
    const DeqConstV dk;
    fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, 0, tid, wave);
    // Every workgroup reads its q rows at the start, all at once (33.5 MB for a 4 x 512-token
    // chunk of 32 heads), so the read is HBM-bound for several us.  When the whole grid runs in
    // one round, the blocks of the lighter half hold their reads back, the lightest longest
    // (a lighter block attends to fewer keys, so it still ends before the heavy ones), and the
    // heavy blocks, which set the launch's length, get their q sooner.
    if (a.q_delay > 0 && n_blk >= 2 && 2 * cblk < n_blk) {
        const int steps = (n_blk / 2 - cblk) * a.q_delay / (n_blk / 2);
        for (int i = 0; i < steps; i++) __builtin_amdgcn_s_sleep(32);  // 2048 clocks each
    }

    // q of this lane's column, read once: the QK norm scale (its q row walked in order), then
    // one power-of-two q scale per workgroup from a bound over all its columns, then the
    // rotation and the hi/lo split from the registers.
    const float ns = QN ? qk_norm_scale(qrow, hdr, L.norm_eps) : 1.0f;
    float q_s, inv_s;
    float xq[NKS][8];
    float2 cs[NKS][4];  // the rotation of each q pair, loaded beside q
    {
        const int qrot = rot_of(L, s, len0 + tok);
        float qb = 0.0f;
#pragma unroll
        for (int t = 0; t < NKS; t++) {
            q_read8(qrow, 2 * t + hf, QN, ns, xq[t], hdr);
            load_rot8(a.rope, a.rope_pairs, 2 * t + hf, qrot, cs[t]);
            // |a cos - b sin| <= |a| + |b|
            qb = fmaxf(qb, fmaxf(fmaxf(fabsf(xq[t][0]) + fabsf(xq[t][1]), fabsf(xq[t][2]) + fabsf(xq[t][3])),
                                 fmaxf(fabsf(xq[t][4]) + fabsf(xq[t][5]), fabsf(xq[t][6]) + fabsf(xq[t][7]))));
        }
        qb = wave_max(qb);
        if (lane == 0) sm_qb[wave] = qb;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) qb = fmaxf(qb, sm_qb[w]);
        q_scale(qb * qmul, q_s, inv_s);
    }
    // q operands of this lane's column: k-step t holds dims 8(2t + hf) .. +7 in f16 (hi); the
    // rest as two fp6 terms per group of 4 k-steps.
    half8 qh[NKS];
    int6v ql1[NG], ql2[NG];
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
                for (int j = 0; j < 8; j++) lo[8 * u + j] = 0.0f;
            }
        }
        q_lo_terms(lo, ql1[g], ql2[g]);
    }
    // Query positions this wave covers (inclusive); qmax < 0 for a wave with no columns.
    const int qmin_w = len0 + c_wave / G;
    const int qmax_w = c_wave < n_cols ? len0 + (min(c_wave + kColsPerWave, n_cols) - 1) / G : -1;
    // (clamped to the capacity: a graph replayed past it reads nothing past it)
    const int key_end = min(len0 + (min(c_blk + COLS, n_cols) - 1) / G + 1, L.P);
    const int n_win = (key_end + kWin - 1) / kWin;

    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) o[db] = (floatx16)0.0f;
    float m_run = 0.0f, l_run = 0.0f;  // m_run: exp2 reference, set by the first window
    bool first = true;

    // Window w+1 is staged into LDS while window w's QK^T runs on the matrix cores (the
    // staging is VALU and LDS-write work); its global loads were issued one iteration earlier.
    stage_codes<HD, NW>(sm, 0, pd, tid, wave, dk);
    stage_scales<HD, NW>(sm, 0, pd, tid, inv_s);
    if (n_win > 1) fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, kWin, tid, wave);
    __syncthreads();

    for (int w = 0; w < n_win; w++) {
        const int buf = w & 1, base = w * kWin;
        const bool more = w + 1 < n_win;
        // QK^T for both 32-key tiles, the two tiles' MFMAs alternating so that no MFMA waits
        // on the one just before it, with the next window's staging in between.  (A wave whose
        // columns all lie before the window computes scores it then drops: on the diagonal
        // only, and it keeps the staging in the MFMAs' basic block.)
        floatx16 sc[2] = {(floatx16)0.0f, (floatx16)0.0f};
        __builtin_amdgcn_s_setprio(3);
        using PD = Pending<HD, NW>;
        constexpr int NPART = PD::SPLIT ? 0 : 8 * PD::NK;  // staging parts, spread over k-steps
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
                // (after the last window this writes the unused buffer)
                if constexpr (NPART > 0) {
#pragma unroll
                    for (int part = t * NPART / NKS; part < (t + 1) * NPART / NKS; part++)
                        stage_part<HD, NW>(sm, buf ^ 1, pd, tid, part, dk);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // the low half of q over these 64 dims: the same codes as fp6
            const int6v k0 = fp6_of(ka0, 1.0f), k1 = fp6_of(ka1, 1.0f);
            sc[0] = mfma_lo6(k0, ql1[g], sc[0], kQlo1E8);
            sc[1] = mfma_lo6(k1, ql1[g], sc[1], kQlo1E8);
            sc[0] = mfma_lo6(k0, ql2[g], sc[0], kQlo2E8);
            sc[1] = mfma_lo6(k1, ql2[g], sc[1], kQlo2E8);
        }
        if constexpr (NPART == 0) stage_codes<HD, NW>(sm, buf ^ 1, pd, tid, wave, dk);
        __builtin_amdgcn_s_setprio(0);
        if (more) stage_scales<HD, NW>(sm, buf ^ 1, pd, tid, inv_s);
        if (w + 2 < n_win) fetch_window<HD, NW>(pd, kbase, vbase, ksb, vsb, base + 2 * kWin, tid, wave);
        if (base <= qmax_w) {
            const bool mask = base + kWin - 1 > qmin_w;  // some key of the window is masked
            window_scores<NDB, SOFTCAP>(sc, sm.sk[buf], sm.svlog[buf], a.softcap, mask, first,
                                        base, hf, qpos, m_run, l_run, o);
            first = false;
            // O^T += V^T P^T one 16-key step at a time: the exps of step st+1 overlap the
            // MFMAs of step st.
#pragma unroll
            for (int st = 0; st < 4; st++) {
                half8 pb, pl;  // p*s_v high and low f16 parts
                step_probs(sc, sm.sv[buf], st, hf, l_run, pb, pl);
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
        float *orow = a.out + (((size_t)s * a.n_tok + tok) * a.n_head + h * G + c % G) * hdr;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int db = 0; db < NDB; db++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float4 v4 = make_float4(o[db][4 * q] * inv, o[db][4 * q + 1] * inv,
                                        o[db][4 * q + 2] * inv, o[db][4 * q + 3] * inv);
                if (32 * db + 8 * q + 4 * hf < hdr) *reinterpret_cast<float4 *>(orow + 32 * db + 8 * q + 4 * hf) = v4;
            }
    }
}

}  // namespace

hipError_t launch_prefill(const KvLayerView &L, const int32_t *d_len, const float *q,
                          int n_head, int n_tok, const float *rope, int rope_pairs,
                          float softcap, float *out, int n_cu, hipStream_t st) {
    PrefillArgs a;
    a.L = L;
    a.len = d_len;
    a.q = q;
    a.rope = rope;
    a.rope_pairs = rope_pairs;
    a.n_head = n_head;
    a.G = n_head / L.H;
    a.n_tok = n_tok;
    a.inv_sqrt_hd = 1.0f / sqrtf((float)L.hdr);
    a.softcap = softcap;
    a.out = out;
    const int n_cols = n_tok * a.G;
    const int cols = kPrefillNW * kColsPerWave;
    const int n_blk = (n_cols + cols - 1) / cols;
    dim3 grid(n_blk, L.H, L.S);
    // (the kernel fits two workgroups per CU below 256 dims, one at 256; measured on config
    // 5's shape: 8 sleep steps for the lightest block, +3.5%)
    const int64_t n_wg = (int64_t)n_blk * L.H * L.S;
    a.q_delay = n_wg <= (int64_t)n_cu * (L.hd > 128 ? 1 : 2) ? 8 : 0;
    const bool cap = softcap > 0.0f, norm = L.qn != nullptr;
#define TS_PF3(HDV, SC, NM, PD)                                                                          \
    {                                                                                                     \
        constexpr size_t lds = sizeof(PrefillLds<HDV>);                                                   \
        if (lds > 64 * 1024)                                                                              \
            (void)hipFuncSetAttribute((const void *)prefill_kernel<HDV, SC, NM, PD>,                      \
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);              \
        prefill_kernel<HDV, SC, NM, PD><<<grid, 64 * kPrefillNW, lds, st>>>(a);                           \
    }
#define TS_PF2(HDV, PD)                                                                                    \
    {                                                                                                     \
        if (cap) { if (norm) TS_PF3(HDV, true, true, PD) else TS_PF3(HDV, true, false, PD) }              \
        else { if (norm) TS_PF3(HDV, false, true, PD) else TS_PF3(HDV, false, false, PD) }                \
    }
#define TS_PF(HDV) { if (L.hdr != L.hd) TS_PF2(HDV, true) else TS_PF2(HDV, false) }
    if (L.hd == 256)
        TS_PF(256)
    else if (L.hd == 128)
        TS_PF(128)
    else if (L.hd == 64)
        TS_PF(64)
    else
        return hipErrorInvalidValue;
#undef TS_PF
#undef TS_PF2
#undef TS_PF3
    return hipGetLastError();
}

}  // namespace ts
