// ts_window.h -- one 64-key window of the INT4 cache against 32 query columns per wave: staging of
// the codes into LDS, q's operands, scores, online softmax and probabilities.  Shared by chunked
// prefill over a cache and attention over a shared prefix.
#pragma once
#include "ts_mfma.h"

namespace ts {

// a b, with 0 for a = 0 and any b.  (The compiler's own operation and not inline asm: a transcendental
// result must not be read by the very next instruction, and the compiler does not see that an asm
// statement reads it; 64-dim rows came out wrong that way.)
__device__ float mul_zero(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

namespace {

constexpr int kPrefillNW = 4;  // waves per workgroup

constexpr int kColsPerWave = 32;
constexpr int kWin = 64;  // keys per window

// Double-buffered window tiles.  K: [key][word] f16 codes; V^T: [dim][8-key group] f16
// codes, each group in the PV operand's key order.  Rows are unpadded; the 16-byte slots
// inside a row are rotated per row (k_slot, v_slot) so that the MFMA operand reads of a wave
// hit distinct LDS banks (chosen by measurement on gfx950: 2x the rate of unrotated rows).
template <int HD>
struct PrefillLds {
    half8 k[2][kWin][HD / 8];
    half8 v[2][HD][kWin / 8];
    float sk[2][kWin], sv[2][kWin];
    float svlog[2];  // log2 of the window's largest s_v
};

// The next window as one thread holds it in flight: its 16-byte pieces of the K window and of
// the V window (NK each; HD=64 with 4 waves has half a piece per thread, so half the threads
// take a K piece and half a V piece) and one scale.
template <int HD, int NW>
struct Pending {
    static constexpr int KCH = kWin * HD / 32;    // 16-byte pieces of the K window (= V window)
    static constexpr int NT = 64 * NW;            // threads
    static constexpr int NK = KCH >= NT ? KCH / NT : 1;
    static constexpr bool SPLIT = KCH < NT;       // threads [0, KCH) take K, [KCH, 2 KCH) take V
    static_assert(KCH % NT == 0 || 2 * KCH == NT, "window pieces must spread evenly");
    uint4 k[NK], v[SPLIT ? 1 : NK];
    float scale;
};

// Slot of word w in the K row of `key`, and of 8-key group sl in the V^T row `row`.
template <int HD>
__device__ inline int k_slot(int key, int w) { return (w + key) & (HD / 8 - 1); }
__device__ inline int v_slot(int row, int sl) { return (sl + (row >> 1)) & 7; }

// Key (within a 32-key tile) that accumulator row R of the QK MFMA stands for.  Lane half h
// holds rows 8q + 4h + r (q, r = 0..3); mapping them to keys 16(q/2) + 8h + 4(q%2) + r gives
// each lane half the 8 consecutive keys 16s + 8h .. +7 of 16-key step s, which is what the PV
// MFMA's B operand wants from it.
__device__ inline int qk_row_key(int R) {
    const int q = R >> 3, h = (R >> 2) & 1, r = R & 3;
    return 16 * (q >> 1) + 8 * h + 4 * (q & 1) + r;
}

// Which 16-byte piece of the window a staging thread owns.  The maps are chosen so that 16
// consecutive lanes write 16 different LDS bank groups:
//  K piece c: chunk k_chunk(c) of the window (the cache's K chunk order, k_word_idx), whose
//  word j is word u of key `key` (k_piece_word); 16 consecutive pieces hold 16 consecutive
//  keys;
//  V piece c: block c / HD, and within it lane group L = c % 64 of the packed layout, its
//  (HD/64)-th piece (c % HD) / 64.
template <int HD>
__device__ inline int k_chunk(int c) {
    if constexpr (HD == 256) {
        const int t = c & 3, n = ((c >> 2) & 3) + 4 * ((c >> 4) & 3), g = (c >> 6) & 3, mh = (c >> 8) & 1;
        return (2 * t + mh) * 64 + 16 * g + n;
    } else if constexpr (HD == 128) {
        const int t = c & 3, n = ((c >> 2) & 3) + 4 * ((c >> 4) & 3), g = (c >> 6) & 3;
        return t * 64 + 16 * g + n;
    } else {
        const int qc = c & 1, n = (c >> 1) & 15, g = (c >> 5) & 3;
        return qc * 64 + 16 * g + n;
    }
}
template <int HD>
__device__ inline void k_piece_word(int c, int j, int &key, int &u) {
    if constexpr (HD == 256) {
        const int t = c & 3, n = ((c >> 2) & 3) + 4 * ((c >> 4) & 3), g = (c >> 6) & 3, mh = (c >> 8) & 1;
        key = 4 * n + t;
        u = 16 * mh + 8 * (j >> 1) + 2 * g + (j & 1);
    } else if constexpr (HD == 128) {
        const int t = c & 3, n = ((c >> 2) & 3) + 4 * ((c >> 4) & 3), g = (c >> 6) & 3;
        key = 4 * n + t;
        u = 8 * (j >> 1) + 2 * g + (j & 1);
    } else {
        const int qc = c & 1, n = (c >> 1) & 15, g = (c >> 5) & 3;
        key = 4 * n + 2 * qc + (j >> 1);
        u = 2 * g + (j & 1);
    }
}
template <int HD>
__device__ inline void v_piece(int cv, int &b, int &piece) {
    constexpr int PPL = HD / 64;  // 16-byte pieces per packed lane group
    b = cv / HD;
    piece = PPL * (cv % 64) + (cv % HD) / 64;
}

template <int HD, int NW>
__device__ inline void fetch_window(Pending<HD, NW> &pd, const uint8_t *kbase, const uint8_t *vbase,
                                    const float *ksb, const float *vsb, int base, int tid, int wave) {
    using P = Pending<HD, NW>;
    constexpr int ROWB = HD / 2;
    auto load_k = [&](int c) {
        return *reinterpret_cast<const uint4 *>(kbase + (size_t)base * ROWB + k_chunk<HD>(c) * 16);
    };
    auto load_v = [&](int c) {
        int b, piece;
        v_piece<HD>(c, b, piece);
        // piece = (HD/64) * ln + t: the t-th 16-byte chunk of lane group ln (v_word_idx)
        constexpr int PPL = HD / 64;
        const int chunk = (piece % PPL) * 64 + piece / PPL;
        return *reinterpret_cast<const uint4 *>(vbase + (size_t)(base / 32 + b) * (HD * 16) + chunk * 16);
    };
    if constexpr (P::SPLIT) {
        // wave-uniform: the first KCH/64 waves take K pieces, the rest V pieces
        if (wave < P::KCH / 64)
            pd.k[0] = load_k(tid);
        else
            pd.k[0] = load_v(tid - P::KCH);
    } else {
#pragma unroll
        for (int i = 0; i < P::NK; i++) pd.k[i] = load_k(tid + P::NT * i);
#pragma unroll
        for (int i = 0; i < P::NK; i++) pd.v[i] = load_v(tid + P::NT * i);
    }
    if (tid < kWin)
        pd.scale = ksb[base + tid];
    else if (tid < 2 * kWin)
        pd.scale = vsb[base + tid - kWin];
}

// Staging of one window's codes, as 8 * NK parts of one 32-bit word each per thread (parts
// [0, 4 NK): K words, [4 NK, 8 NK): V words), so the caller can spread them over other work.
// Only for the layout where every thread holds NK K pieces and NK V pieces (!SPLIT).
template <int HD, int NW, class SM>
__device__ inline void stage_part(SM &sm, int buf, const Pending<HD, NW> &pd, int tid,
                                  int part, const DeqConst &dk) {
    using P = Pending<HD, NW>;
    static_assert(!P::SPLIT, "per-part staging needs whole K and V pieces per thread");
    const int i = (part % (4 * P::NK)) / 4, j = part % 4;
    const int c = tid + P::NT * i;
    if (part < 4 * P::NK) {
        const uint4 &x = pd.k[i];
        const uint32_t wj = j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w;
        int key, u;
        k_piece_word<HD>(c, j, key, u);
        sm.k[buf][key][k_slot<HD>(key, u)] = dequant8_c(wj, dk);
    } else {
        // V: lane L holds 4 words of packed lane group ln = L (key group g = ln/16, dim row dl
        // = ln%16); lane L^16 holds the same words of key group g^1.  Words of groups 2p and
        // 2p+1 hold keys 8p..8p+7 in their low halves (nibbles 0-3) and 16+8p..16+8p+7 in
        // their high halves, so the even lane builds the dword of low halves, the odd lane the
        // one of high halves: one 8-key group of the V^T row each.
        const uint4 &x = pd.v[i];
        const uint32_t wj = j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w;
        int b, piece;
        v_piece<HD>(c, b, piece);
        const int ln = c % 64, dl = ln & 15, odd = (ln >> 4) & 1, pair = ln >> 5;
        const int td0 = (c % HD) / 64 * 4;
        const int sl = 4 * b + 2 * odd + pair;
        // byte selects of v_perm_b32(pw, w): even lanes low(w) | low(pw) << 16, odd lanes
        // high(pw) | high(w) << 16 (one instruction, no lane-divergent branch)
        const uint32_t sel = odd ? 0x03020706u : 0x05040100u;
        const uint32_t pw = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (threadIdx.x ^ 16), (int)wj);
        const uint32_t d = __builtin_amdgcn_perm(pw, wj, sel);
        const int row = 16 * (td0 + j) + dl;
        sm.v[buf][row][v_slot(row, sl)] = dequant8_c(d, dk);
    }
}

// All of one window's codes into LDS.
template <int HD, int NW, class SM>
__device__ inline void stage_codes(SM &sm, int buf, const Pending<HD, NW> &pd, int tid,
                                   int wave, const DeqConst &dk) {
    using P = Pending<HD, NW>;
    if constexpr (P::SPLIT) {
        // V staging as in stage_part, for a thread that holds one V piece
        auto put_k = [&](int c, const uint4 &x) {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int key, u;
                k_piece_word<HD>(c, j, key, u);
                sm.k[buf][key][k_slot<HD>(key, u)] = dequant8_c(w[j], dk);
            }
        };
        auto put_v = [&](int c, const uint4 &x) {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            int b, piece;
            v_piece<HD>(c, b, piece);
            const int ln = c % 64, dl = ln & 15, odd = (ln >> 4) & 1, pair = ln >> 5;
            const int td0 = (c % HD) / 64 * 4;
            const int sl = 4 * b + 2 * odd + pair;
            const uint32_t sel = odd ? 0x03020706u : 0x05040100u;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t pw = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (threadIdx.x ^ 16), (int)w[j]);
                const uint32_t d = __builtin_amdgcn_perm(pw, w[j], sel);
                const int row = 16 * (td0 + j) + dl;
                sm.v[buf][row][v_slot(row, sl)] = dequant8_c(d, dk);
            }
        };
        if (wave < P::KCH / 64)
            put_k(tid, pd.k[0]);
        else
            put_v(tid - P::KCH, pd.k[0]);
    } else {
#pragma unroll
        for (int part = 0; part < 8 * P::NK; part++) stage_part<HD, NW, SM>(sm, buf, pd, tid, part, dk);
    }
}

// The window's scales into LDS (kept apart from the code staging, which is branch-free so it
// can be scheduled in between the QK matrix-core instructions).
// ANY: a scale may be infinite or NaN at keys that no column sees (what a shortened sequence left
// behind): the bound on p s_v is then taken over the others.
template <int HD, int NW, bool ANY = false, class SM>
__device__ inline void stage_scales(SM &sm, int buf, const Pending<HD, NW> &pd, int tid,
                                    float inv_s) {
    if (tid < kWin) {
        sm.sk[buf][tid] = pd.scale * inv_s;  // undo the q operand scale (a power of two: exact)
    } else if (tid < 2 * kWin) {
        sm.sv[buf][tid - kWin] = pd.scale;
        // (one whole wave: threads kWin .. 2 kWin - 1; the scales are >= 0)
        const float m = wave_max_nonneg(ANY ? (pd.scale < INFINITY ? pd.scale : 0.0f) : pd.scale);
        if (tid == kWin) sm.svlog[buf] = __log2f(m);
    }
}

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int int6v __attribute__((ext_vector_type(6)));
typedef int int8v __attribute__((ext_vector_type(8)));
typedef _Float16 half32 __attribute__((ext_vector_type(32)));
typedef float float32v __attribute__((ext_vector_type(32)));

// q's low half on the fp6 matrix-core path.  The low half q - f16(q) needs only a few bits of
// its own: it enters v_mfma_scale_f32_32x32x64_f8f6f4 as fp6 e2m3 (3 mantissa bits, largest
// 7.5) with a power-of-two scale, while the K codes on the other side (integers -7..7) are
// exact in e2m3.  That MFMA does 64 k-steps of 32x32 in about the time of one 32x32x16 f16
// MFMA (a quarter of the four f16 MFMAs it replaces); two terms (the second one the rounding
// rest of the first) keep q to about f16 hi + lo accuracy.
__device__ inline float exp2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// 4 k-steps of an f16 operand (32 values per lane, in operand order) as fp6 divided by s.
__device__ inline int6v fp6_of(const half8 (&x)[4], float s) {
    half32 v;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) v[8 * u + j] = x[u][j];
    return __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(v, s);
}

// o += a b^T over 64 k-steps, a: fp6 codes (scale 1), b: fp6 with scale 2^(e8 - 127).
__device__ inline floatx16 mfma_lo6(int6v a, int6v b, floatx16 c, int e8) {
    const int8v a8 = {a[0], a[1], a[2], a[3], a[4], a[5], 0, 0};
    const int8v b8 = {b[0], b[1], b[2], b[3], b[4], b[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 2, 2, 0, 127, 0, e8);
}

// q's low half over one group of 4 k-steps (32 values lo[], f32) as two fp6 terms with fixed
// scales: q is scaled so that |q| < 2^14 (q_scale), so its f16 high half leaves |lo| <= 4
// (half an f16 ulp at 2^13); t1 = fp6(lo) rounds that to within 0.125, and t2 = fp6((lo - t1)
// / 2^-5) keeps the rest to 2^-8: q to ~2^-22 of its bound, as a second f16 half would.
constexpr int kQlo1E8 = 127, kQlo2E8 = 127 - 5;
__device__ inline void q_lo_terms(const float (&lo)[32], int6v &t1, int6v &t2) {
    floatx16 a, b;
#pragma unroll
    for (int i = 0; i < 16; i++) {  // the conversion interleaves its two sources
        a[i] = lo[2 * i];
        b[i] = lo[2 * i + 1];
    }
    t1 = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, 1.0f);
    const float32v back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(t1, 1.0f);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        a[i] = lo[2 * i] - back[2 * i];
        b[i] = lo[2 * i + 1] - back[2 * i + 1];
    }
    t2 = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, exp2i(-5));
}

// split_q8 with the low half kept in f32 (the fp6 terms are taken from it).
__device__ inline void split_q8_f32(float (&x)[8], const float2 (&cs)[4], int u, int rope_pairs, float mul,
                                    half8 &hi, float *lo) {
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (4 * u + i < rope_pairs) rope_rotate(x[2 * i], x[2 * i + 1], cs[i]);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = opaque(x[kPerm[j]] * mul);
        const _Float16 h = (_Float16)v;
        hi[j] = h;
        lo[j] = v - (float)h;
    }
}

// Max / sum over the two lane halves (lanes l and l^32) that hold one column.
__device__ inline float half_max(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float half_sum(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Scores of one 64-key window for this lane's column, in place (sc[kb][4q + r] is key
// 32kb + qk_row_key(8q + 4h + r)), left relative to the running reference m_run:
// sc = x s_k - m_run (one FMA per score; softcap in between when on), causal mask, then the
// online-softmax state update.  The reference is raised only when the window breaks
// p <= 2^8 or p*s_v <= 2^15 (f16 range), and the scores move down with it; the first window
// (first, uniform; m_run = 0 and nothing accumulated yet) sets it from its own max.
template <int NDB, bool SOFTCAP>
__device__ inline void window_scores(floatx16 (&sc)[2], const float *sk, float svl, float softcap,
                                     bool mask, bool first, int base, int h, int qpos, float &m_run,
                                     float &l_run, floatx16 (&o)[NDB]) {
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const floatx4 sk4 = *reinterpret_cast<const floatx4 *>(sk + 32 * kb + 16 * (q >> 1) + 8 * h + 4 * (q & 1));
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float x;
                if constexpr (SOFTCAP) {
                    x = sc[kb][4 * q + r] * sk4[r];
                    x = tanhf(x / softcap) * softcap * kLog2e - m_run;
                } else {
                    x = __builtin_fmaf(sc[kb][4 * q + r], sk4[r], -m_run);
                }
                sc[kb][4 * q + r] = x;
            }
        }
    }
    if (mask) {
        // a real branch: only windows on the causal diagonal pay for the compares
        asm volatile("");
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (base + 32 * kb + 16 * (q >> 1) + 8 * h + 4 * (q & 1) + r > qpos) sc[kb][4 * q + r] = -INFINITY;
    }
    float mloc = kMinit;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int i = 0; i < 16; i++) mloc = fmaxf(mloc, sc[kb][i]);
    mloc = half_max(mloc);
    const float need = fmaxf(mloc - 8.0f, mloc + svl - 15.0f);  // relative to m_run
    if (__builtin_amdgcn_ballot_w64(first || need > 0.0f) != 0) {
        const float delta = (first || need > 0.0f) ? mloc + fmaxf(0.0f, svl - 15.0f) : 0.0f;
        if (!first) {
            const float alpha = exp2f(-delta);
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; db++) o[db] *= alpha;
        }
        m_run += delta;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[kb][i] = sc[kb][i] - delta;
    }
}

// Probabilities of 16-key step st (keys 16st + 8h + 0..7 of the window) times s_v, split
// hi + lo in f16 in the PV operand's slot order; adds the p to l_run.  p*s_v = hi + lo keeps
// ~22 bits: one f16 would carry a relative error of 2^-11 into the output whenever a few
// keys dominate the row.
// ANY: as stage_scales; the product with a hidden key's p = 0 is 0 whatever s_v is.
template <bool ANY = false>
__device__ inline void step_probs(const floatx16 (&sc)[2], const float *sv, int st, int h,
                                  float &l_run, half8 &pb, half8 &pl) {
    const int kb = st >> 1;
#pragma unroll
    for (int qq = 0; qq < 2; qq++) {
        const int q = 2 * (st & 1) + qq;
        const floatx4 sv4 = *reinterpret_cast<const floatx4 *>(sv + 32 * kb + 16 * (q >> 1) + 8 * h + 4 * (q & 1));
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float p = __builtin_amdgcn_exp2f(sc[kb][4 * q + r]);  // sc is relative
            l_run += p;
            // hi: the exact product p s_v rounded once to f16; lo: the exact remainder
            // p s_v - hi rounded once (both one fused multiply-add with an f16 result)
            // key 16st + 8h + 4(q&1) + r: slot 2r + (q&1)
            if constexpr (ANY) {
                const float w = opaque(mul_zero(p, sv4[r]));
                const _Float16 hi = (_Float16)w;
                pb[2 * r + (q & 1)] = hi;
                pl[2 * r + (q & 1)] = (_Float16)(w - (float)hi);
            } else {
                const _Float16 hi = (_Float16)__builtin_fmaf(p, sv4[r], 0.0f);
                pb[2 * r + (q & 1)] = hi;
                pl[2 * r + (q & 1)] = (_Float16)__builtin_fmaf(p, sv4[r], -(float)hi);
            }
        }
    }
}

}  // namespace
}  // namespace ts
