// ts_decode_split.h -- one split of the 16x16 decode kernel: a workgroup's part of one (sequence, kv head)
// stream.  Shared by the decode launches and by attention behind a shared prefix, whose launch
// holds such workgroups beside those over the prefix.
#pragma once
#include "ts_mfma.h"

namespace ts {
namespace {

struct DecodeArgs {
    KvLayerView L;
    const int32_t *len;
    // hlen >= 0 (one sequence): its length, given by the host with the launch (as the
    // reference passes its uniforms) instead of read from len[] first: an eager call whose
    // host length is known to match the device's.  -1: read len[].
    int hlen;
    const float *q;
    const float *rope;
    int rope_pairs;
    int n_head;
    int G;   // query heads per workgroup: n_head / n_kv (integer kernel, up to 16), at most 8 per
             // group (16x16 kernel)
    int Gt;  // query heads per kv head (n_head / n_kv)
    int NG;  // head groups per kv head: grid.y = n_kv * NG (integer kernel: 1)
    int chunk;
    int n_split;  // grid.x: the last split of a sequence runs to its end
    float inv_sqrt_hd;
    float softcap;
    float *out;
    float *ws;  // partial o [S][n_head][n_split][hd], then m [..][n_split], l [..][n_split]

    // Fused append (ts_attn_decode_append): the new token's raw K and V, [S][H][hd], or null.
    const float *k_new, *v_new;

    // ts_attn_decode_append_advance: the lengths to advance by one (the array len points to)
    // and the arrival counter of the kernel that does it, or null.
    int32_t *adv_len;
    int32_t *adv_ctr;
};

// Every workgroup of the launch's last kernel calls this once, after its last read of the
// lengths: the workgroup that arrives last (all others have read them by then) advances every
// length by one and clears the counter for the next launch.  Call from all threads of the
// workgroup (the barrier orders this workgroup's length reads before its arrival).
__device__ inline void arrive_and_advance(const DecodeArgs &a) {
    if (!a.adv_ctr) return;
    if (a.hlen >= 0) {
        // the length came with the launch and no workgroup reads len[]: one plain store of the
        // advanced value, no arrival count (a returning atomic's round trip saved)
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) a.adv_len[0] = a.hlen + 1;
        return;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int n_wg = gridDim.x * gridDim.y * gridDim.z;
        if (atomicAdd(a.adv_ctr, 1) == n_wg - 1) {
            for (int s = 0; s < a.L.S; s++) a.adv_len[s] += 1;
            *a.adv_ctr = 0;
        }
    }
}

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// One 64-position window of one (sequence, kv head) stream, as held by one lane in registers
// while it is in flight: K rows (tile kt, row n, the words of lane group g), V blocks (block b,
// words lane*NTD..), and one K and one V scale (position base + lane).
template <int HD>
struct Window {
    static constexpr int WPG = HD / 32, NTD = HD / 16;
    uint32_t kw[4][WPG];
    uint32_t vw[2][NTD];
    float sk, sv;
};

// Buffer resources of one (sequence, kv head) stream, bounded to the positions of one split:
// loads past the bound return zeros without touching memory, so prefetches can be issued
// unconditionally (which keeps the compiler's load counters static, so the wait before each
// window only covers that window's own loads).
struct Streams {
    __amdgpu_buffer_rsrc_t k, v;
    const float *ksb, *vsb;
    int last;  // last position of the split
};

__device__ inline __amdgpu_buffer_rsrc_t make_rsrc(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000);
}

// K word that lane group g feeds to the 16x16 QK instruction at k-step t (of the WPG words of
// its row): the words the cache keeps together in one chunk for that row and group (the
// chunk order of k_word_idx), so one load per row brings them all.
template <int HD>
__device__ inline int k16_word(int g, int t) {
    if constexpr (HD >= 128) return 8 * (t >> 1) + 2 * g + (t & 1);
    else return 2 * g + t;
}

template <int HD>
__device__ __forceinline__ void load_window(Window<HD> &w, const Streams &st, int base, int n,
                                            int g, int lane) {
    constexpr int WPG = HD / 32, NTD = HD / 16, ROWB = HD / 2;
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
        // row r = 16 kt + n of the window: words k16_word(g, 0..WPG-1) sit in chunk
        // ((r % 4) / (128 / HD)) * 64 + 16 g + r / 4, at word (r % 2) * 2 for hd 64
        const int r = 16 * kt + n;
        if constexpr (WPG == 8) {
            // hd 256: the 8 words sit in chunks (2 (r % 4) + c) * 64 + 16 g + r / 4, c = 0, 1
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int koff = ((2 * (r & 3) + c) * 64 + 16 * g + (r >> 2)) * 16;
                const u32x4 t4 = __builtin_amdgcn_raw_buffer_load_b128(st.k, koff, base * ROWB, 0);
                w.kw[kt][4 * c] = t4[0]; w.kw[kt][4 * c + 1] = t4[1]; w.kw[kt][4 * c + 2] = t4[2]; w.kw[kt][4 * c + 3] = t4[3];
            }
        } else if constexpr (WPG == 4) {
            const int koff = ((r & 3) * 64 + 16 * g + (r >> 2)) * 16;
            const u32x4 t4 = __builtin_amdgcn_raw_buffer_load_b128(st.k, koff, base * ROWB, 0);
            w.kw[kt][0] = t4[0]; w.kw[kt][1] = t4[1]; w.kw[kt][2] = t4[2]; w.kw[kt][3] = t4[3];
        } else {
            const int koff = (((r & 3) >> 1) * 64 + 16 * g + (r >> 2)) * 16 + 8 * (r & 1);
            const u32x2 t2 = __builtin_amdgcn_raw_buffer_load_b64(st.k, koff, base * ROWB, 0);
            w.kw[kt][0] = t2[0]; w.kw[kt][1] = t2[1];
        }
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
        for (int q4 = 0; q4 < NTD / 4; q4++) {
            // words 4 q4 .. 4 q4 + 3 of lane group `lane`: chunk q4 * 64 + lane
            const u32x4 t4 = __builtin_amdgcn_raw_buffer_load_b128(st.v, (q4 * 64 + lane) * 16 + b * (HD * 16), (base / 32) * (HD * 16), 0);
            w.vw[b][4 * q4 + 0] = t4[0]; w.vw[b][4 * q4 + 1] = t4[1];
            w.vw[b][4 * q4 + 2] = t4[2]; w.vw[b][4 * q4 + 3] = t4[3];
        }
    }
    // Scales: plain loads with the index clamped into the split; windows past the end re-read
    // valid, unused scales.
    const int sp = min(base + lane, st.last);
    w.sk = st.ksb[sp];
    w.sv = st.vsb[sp];
}

// Running state of one wave: O^T accumulators (column n = head, rows = dims 16td+4g+r), the
// reference exponent m (exp2 domain) and the softmax sum l.
template <int HD>
struct WaveState {
    floatx4 o[HD / 16];
    float m, l;
};

// q operands in LDS, [k-step t][lane], shared by the waves of a workgroup.  Column n of the
// MFMA (lane group n = lane & 15) carries the f16 high part of head n for n < G and the low
// part (q - hi) of head n - G for G <= n < 2G, so one MFMA computes both halves of every
// score; G <= 8 keeps 2G within the 16 columns.
template <int HD>
struct QLds {
    half8 p[HD / 32][64];
};

// live: this lane's column carries a head (n < 2G); lo_col: it carries the low parts (G <= n);
// partner4: byte address (for ds_bpermute) of the lane holding the other part of its scores.
template <int HD, bool SOFTCAP>
__device__ __forceinline__ void process_window(const Window<HD> &w, WaveState<HD> &st,
                                               const QLds<HD> &qs, float *stage, int base, int end,
                                               int lane, int g, bool live, bool lo_col, int partner4,
                                               float inv_s, float softcap, const DeqConst &dc) {
    constexpr int WPG = HD / 32, NTD = HD / 16;
    // Scales: one per lane in registers -> this wave's LDS stage -> the 4 positions each lane
    // holds per tile (16kt + 4g + r).  Same-wave LDS traffic is ordered: no barrier needed.
    stage[lane] = w.sk * inv_s;  // undo the q operand scale (a power of two: exact)
    stage[64 + lane] = w.sv;
    // ---- S^T = K Q^T (rows: positions, columns: heads), hi + lo q in one accumulator --------
    floatx4 sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; kt++) sc[kt] = (floatx4)0.0f;
#pragma unroll
    for (int t = 0; t < WPG; t++) {
        const half8 qp = qs.p[t][lane];
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            const half8 ka = dequant8(w.kw[kt][t], dc);
            sc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qp, sc[kt], 0, 0, 0);
        }
    }
    // hi column + lo column: lanes n and n +- G swap partial scores and both hold the same sum
    // (a + b == b + a exactly), so the two columns run identical softmax arithmetic below.
#pragma unroll
    for (int kt = 0; kt < 4; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            sc[kt][r] += __int_as_float(__builtin_amdgcn_ds_bpermute(partner4, __float_as_int(sc[kt][r])));
    // ---- softmax ----------------------------------------------------------------------------
    // x = score * log2(e).  s_v is folded into the probabilities: P = 2^(x - m) * s_v, with the
    // window reference m >= max(x) + log2(max s_v), so P <= 1 always fits f16.
    float x[16], sv[16];
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
        const floatx4 sk4 = *reinterpret_cast<const floatx4 *>(stage + 16 * kt + 4 * g);
        const floatx4 sv4 = *reinterpret_cast<const floatx4 *>(stage + 64 + 16 * kt + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float v = sc[kt][r] * sk4[r];
            if constexpr (SOFTCAP) v = tanhf(v * (1.0f / kLog2e) / softcap) * softcap * kLog2e;
            x[4 * kt + r] = v;
            sv[4 * kt + r] = sv4[r];
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {  // positions past the split's end
        const int pos = base + 16 * (i >> 2) + 4 * g + (i & 3);
        if (pos >= end) {
            x[i] = -INFINITY;
            sv[i] = 0.0f;
        }
    }
    float xm = x[0], sm = sv[0];
#pragma unroll
    for (int i = 1; i < 16; i++) {
        xm = fmaxf(xm, x[i]);
        sm = fmaxf(sm, sv[i]);
    }
    xm = group_max(xm);
    sm = group_max(sm);
    float mw = xm + __builtin_amdgcn_logf(sm);
    mw = fminf(fmaxf(mw, xm - 64.0f), xm + 64.0f);
    // Rescale only when the reference would grow by more than 2^8; in between P stays below
    // 2^8 (fine for f16) and no accumulator is touched.
    if (__any(live && mw > st.m + 8.0f)) {
        asm volatile("" ::: "memory");  // keep this a branch: the multiply is the rare case
        const float m_new = fmaxf(st.m, mw);
        const float alpha = fast_exp2(st.m - m_new);
        st.l *= alpha;
#pragma unroll
        for (int td = 0; td < NTD; td++) st.o[td] *= alpha;
        st.m = m_new;
    }
    float psum = 0.0f, pv[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float p = fast_exp2(x[i] - st.m);
        psum += p;
        pv[i] = p * sv[i];
    }
    st.l += psum;
    // ---- O^T += V^T P^T ---------------------------------------------------------------------
    // P = hi + lo in f16 (~22 bits, like q): the hi columns feed f16(P), the lo columns
    // P - f16(P); a single f16 P would carry a relative error of 2^-11 straight into the output
    // whenever one position dominates the softmax.  Columns past 2G hold finite garbage that
    // only feeds output columns never read.
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float hi = split_hi(pv[i]);
        pv[i] = lo_col ? pv[i] - hi : hi;
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
        half8 pb;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            // slots (2r, 2r+1) = positions 4g+r of tiles 2b and 2b+1
            const half2_t pr = {(_Float16)pv[4 * (2 * b) + r], (_Float16)pv[4 * (2 * b + 1) + r]};
            pb[2 * r] = pr[0];
            pb[2 * r + 1] = pr[1];
        }
#pragma unroll
        for (int td = 0; td < NTD; td++) {
            const half8 va = dequant8(w.vw[b][td], dc);
            st.o[td] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, st.o[td], 0, 0, 0);
        }
    }
}

// Fused append, run by one wave of the workgroup whose split holds position p = len[s]: the
// quantize-on-append of ts_append.hip for one (sequence, kv head) and one position, with the
// same arithmetic (ts_quant.h), so codes and scales are bit-identical.  Lane i owns the
// rotation pairs i + 64 j (j < PPL: one pair per lane up to head dim 128, two at 256), i.e.
// dims 2(i + 64j) and +1.  Writes the K row, both scales and the position's nibble of every V
// word (read-modify-write: only this workgroup touches the block), and leaves the dequantized
// row ((code - 8) * scale, the values the cache now holds) in kd / vd.
//
// Two phases, so a caller can issue every load of the append together (one memory round trip)
// before anything else: append_load, then append_store.
template <int HD>
struct AppendIn {
    static constexpr int PPL = HD > 128 ? 2 : 1;
    float k[PPL][2], v[PPL][2];  // raw new K / V of the lane's pairs
    float2 cs[PPL];              // rotation of each pair at the position's rotation position
    float kn[PPL][2];            // K norm weights of the pairs' dims (QK norm)
    uint32_t vold[PPL][2];       // the V words holding the pairs' dims at this position
};

template <int HD, bool NORM>
__device__ __forceinline__ void append_load(const DecodeArgs &a, int s, int h, int p, int lane, AppendIn<HD> &in,
                                            int hdr) {
    constexpr int PPL = AppendIn<HD>::PPL;
    const KvLayerView &L = a.L;
    const size_t row = (size_t)s * L.H + h;
    const int pr = rot_of(L, s, p);
    const int q = p & 31, gq = (q & 15) >> 2;
    const uint32_t *vb = reinterpret_cast<const uint32_t *>(L.vp + (row * (L.P / 32) + (p >> 5)) * (HD * 16));
#pragma unroll
    for (int j = 0; j < PPL; j++) {
        const int i = lane + 64 * j;
        const bool on = i < HD / 2;
        // rows of hdr floats; the stored dims past them are 0 (their lanes load the row's
        // first pair, unconditionally, and drop it)
        const bool dim_in = on && 2 * i < hdr;
        const size_t src = row * hdr + 2 * (dim_in ? i : 0);
        const float2 kk = *reinterpret_cast<const float2 *>(a.k_new + src);
        const float2 vv = *reinterpret_cast<const float2 *>(a.v_new + src);
        in.k[j][0] = dim_in ? kk.x : 0.f; in.k[j][1] = dim_in ? kk.y : 0.f;
        in.v[j][0] = dim_in ? vv.x : 0.f; in.v[j][1] = dim_in ? vv.y : 0.f;
        const int ir = i < a.rope_pairs ? i : 0;
        in.cs[j] = *reinterpret_cast<const float2 *>(a.rope + ((size_t)pr * a.rope_pairs + ir) * 2);
        in.kn[j][0] = NORM && L.kn && dim_in ? L.kn[2 * i] : 1.0f;
        in.kn[j][1] = NORM && L.kn && dim_in ? L.kn[2 * i + 1] : 1.0f;
        const int ic = on ? i : 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int d = 2 * ic + e;
            in.vold[j][e] = vb[v_word_idx(gq * 16 + (d & 15), d >> 4)];
        }
    }
}

// write = false: only the dequantized rows (a head group other than the first, whose
// workgroup quantizes the same row for its own heads' scores).
template <int HD, bool NORM>
__device__ void append_store(const DecodeArgs &a, int s, int h, int p, int lane, const AppendIn<HD> &in,
                             float *kd, float *vd, int hdr, bool write = true) {
    constexpr int ROWB = HD / 2, PPL = AppendIn<HD>::PPL;
    const KvLayerView &L = a.L;
    const bool KN = NORM && L.kn != nullptr;  // QK norm of K
    const size_t row = (size_t)s * L.H + h;
    float k[PPL][2], v[PPL][2];
#pragma unroll
    for (int j = 0; j < PPL; j++) {
        k[j][0] = in.k[j][0]; k[j][1] = in.k[j][1];
        v[j][0] = in.v[j][0]; v[j][1] = in.v[j][1];
    }
    // QK norm scale of the new K row: its squares summed in dimension order across the lanes
    // (pairs 0..63, then 64..127)
    float ns = 0.0f;
    if (KN) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PPL; j++)
            sum = ordered_sum_pairs(sq_rn(k[j][0]), sq_rn(k[j][1]), HD / 2 < 64 ? HD / 2 : 64, sum);
        ns = qk_norm_scale_from_sum(sum, hdr, L.norm_eps);
    }
    float km = 0.0f, vm = 0.0f;
#pragma unroll
    for (int j = 0; j < PPL; j++) {
        const int i = lane + 64 * j;
        if (i < HD / 2) {
            if (KN) {
                k[j][0] = qk_norm_apply(k[j][0], ns, in.kn[j][0]);
                k[j][1] = qk_norm_apply(k[j][1], ns, in.kn[j][1]);
            }
            if (i < a.rope_pairs) rope_rotate(k[j][0], k[j][1], in.cs[j]);
        }
        km = fmaxf(km, fmaxf(fabsf(k[j][0]), fabsf(k[j][1])));
        vm = fmaxf(vm, fmaxf(fabsf(v[j][0]), fabsf(v[j][1])));
    }
    const float ks = quant_scale(wave_max(km));
    const float vs = quant_scale(wave_max(vm));
    if (write && lane == 0) {
        L.ks[row * L.P + p] = ks;
        L.vs[row * L.P + p] = vs;
    }
    // V block p/32: dim d of key group gq sits in word v_word_idx(gq*16 + d%16, d/16), position
    // 4gq + r of tile t at nibble r + 4t.
    const int q = p & 31, t = q >> 4, gq = (q & 15) >> 2, nib = (q & 3) + 4 * t;
    uint32_t *vb = reinterpret_cast<uint32_t *>(L.vp + (row * (L.P / 32) + (p >> 5)) * (HD * 16));
#pragma unroll
    for (int j = 0; j < PPL; j++) {
        const int i = lane + 64 * j;
        const bool on = i < HD / 2;
        const uint32_t c0 = encode(k[j][0], ks), c1 = encode(k[j][1], ks);
        const uint32_t e0 = encode(v[j][0], vs), e1 = encode(v[j][1], vs);
        // K row: word u holds dims 8u..8u+7 at bits 4*(d - 8u); pairs 4u..4u+3 share word u.
        uint32_t kw = on ? (c0 | (c1 << 4)) << (8 * (i & 3)) : 0u;
        kw |= __shfl_xor(kw, 1, 64);
        kw |= __shfl_xor(kw, 2, 64);
        if (write && on && (i & 3) == 0)
            reinterpret_cast<uint32_t *>(L.kp + row * L.P * ROWB)[k_word_idx<HD>(p, i >> 2)] = kw;
        if (on) {
            if (write) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = 2 * i + e;
                    vb[v_word_idx(gq * 16 + (d & 15), d >> 4)] =
                        (in.vold[j][e] & ~(0xFu << (4 * nib))) | ((e ? e1 : e0) << (4 * nib));
                }
            }
            kd[2 * i] = (float)((int)c0 - 8) * ks;
            kd[2 * i + 1] = (float)((int)c1 - 8) * ks;
            vd[2 * i] = (float)((int)e0 - 8) * vs;
            vd[2 * i + 1] = (float)((int)e1 - 8) * vs;
        }
    }
}

// Scores of the new position (dequantized row kd, in this wave's LDS) for the G query heads
// hb .. hb + G - 1 of sequence s, in the exp2 domain, from the rotated f32 q (as load_q8
// rotates it); one wave.  qp[hh][j]: dims 2(i + 64j), +1 of head hh's raw q, cs[j]: the
// rotation of that pair at the query's rotation position.
template <int HD, bool SOFTCAP, bool NORM, int GMAX>
__device__ void new_token_scores(const DecodeArgs &a, int s, int hb, int G, int lane,
                                 const float2 (&qp)[GMAX][AppendIn<HD>::PPL], const float2 (&cs)[AppendIn<HD>::PPL],
                                 const float *kd, float *xnew, int hdr) {
    constexpr int PPL = AppendIn<HD>::PPL;
    const float *const QN = NORM ? a.L.qn : nullptr;
    const float *qg = a.q + ((size_t)s * a.n_head + hb) * hdr;
    float nhs[GMAX];
    if (QN) q_norm_scales_wave<HD, GMAX>(qg, G, a.L.norm_eps, hdr, nhs);
    // (a guard, not a break: the loop unrolls fully, so qp stays in registers)
#pragma unroll
    for (int hh = 0; hh < GMAX; hh++) {
        if (hh >= G) continue;
        const float nh = QN ? nhs[hh] : 1.0f;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < PPL; j++) {
            const int i = lane + 64 * j;
            float q0 = qp[hh][j].x, q1 = qp[hh][j].y;
            if (QN && 2 * i < hdr) {
                q0 = qk_norm_apply(q0, nh, QN[2 * i]);
                q1 = qk_norm_apply(q1, nh, QN[2 * i + 1]);
            }
            if (i < a.rope_pairs) rope_rotate(q0, q1, cs[j]);
            dot += i < HD / 2 ? q0 * kd[2 * i] + q1 * kd[2 * i + 1] : 0.0f;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) dot += __shfl_xor(dot, o, 64);
        float x = dot * a.inv_sqrt_hd;
        if constexpr (SOFTCAP) x = tanhf(x / a.softcap) * a.softcap;
        if (lane == 0) xnew[hh] = x * kLog2e;
    }
}

// The raw q pairs new_token_scores takes: dims 2(i + 64j), +1 of query heads hb .. hb + G - 1.
template <int HD, int GMAX>
__device__ __forceinline__ void load_q_pairs(const DecodeArgs &a, int s, int hb, int G, int lane,
                                             float2 (&qp)[GMAX][AppendIn<HD>::PPL], int hdr) {
    const float *qg = a.q + ((size_t)s * a.n_head + hb) * hdr;
#pragma unroll
    for (int hh = 0; hh < GMAX; hh++)
#pragma unroll
        for (int j = 0; j < AppendIn<HD>::PPL; j++) {
            const int i = lane + 64 * j;
            const bool use = hh < G && i < HD / 2 && 2 * i < hdr;
            const float2 t = *reinterpret_cast<const float2 *>(qg + (size_t)(hh < G ? hh : 0) * hdr + 2 * (use ? i : 0));
            qp[hh][j] = make_float2(use ? t.x : 0.f, use ? t.y : 0.f);
        }
}

// Split partial of one head: unnormalized o (dim d), and with d == 0 the reference exponent m
// and the sum l, for decode_combine_kernel.
__device__ inline void store_partial(const DecodeArgs &a, size_t head, int split, int HD, int d, float acc,
                                     float M, float lsum) {
    const size_t rows = (size_t)a.L.S * a.n_head * a.n_split, r = head * a.n_split + split;
    a.ws[r * HD + d] = acc;
    if (d == 0) {
        a.ws[rows * HD + r] = M;
        a.ws[rows * (HD + 1) + r] = lsum;
    }
}

// LDS: q operands, per-wave scale stages; and the merge area, apart from them so that a
// wave writes its share of the merge as soon as its windows are done.
template <int HD, int NW>
struct DecodeSplitSmem {
    static constexpr int OST = HD + 4;  // 16-byte rows of the merge area
    struct {
        QLds<HD> q;
        float stage[NW][128];
    } run;
    struct {
        __align__(16) float o[NW][16 * OST];
        float m[NW][8], l[NW][8];
    } merge;
};

// split, by, seq: the workgroup's split, (kv head, head group) and sequence; PAD, NW as in
// decode_split_kernel.  The partials are the caller's to join.  LDS: sm; kd, vd [HD] and xnew [8], the fused append's dequantized new K and V rows
// and its score per head.
template <int HD, bool SOFTCAP, bool NORM, bool PAD, int NW>
__device__ __forceinline__ void decode_split(const DecodeArgs &a, int split_x, int by, int seq, DecodeSplitSmem<HD, NW> &sm,
                                             float *kd, float *vd, float *xnew) {
#define TS_SPLIT_X split_x
#define TS_SPLIT_Y by
#define TS_SPLIT_Z seq
#define TS_SPLIT_LDS
#define TS_SPLIT_KEEP true
#include "ts_decode_split_body.h"
#undef TS_SPLIT_X
#undef TS_SPLIT_Y
#undef TS_SPLIT_Z
#undef TS_SPLIT_LDS
#undef TS_SPLIT_KEEP
}

}  // namespace
}  // namespace ts
