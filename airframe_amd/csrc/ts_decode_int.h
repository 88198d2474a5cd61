// ts_decode_int.h -- the integer decode kernel (G <= 16 query heads per kv head), the merge of splits, and their
// launches.  Shared by the decode launches and by attention that adds up what every slot receives, which
// also wants each score (SCORES).
#pragma once
#include "ts_decode_split.h"
#include "ts_quant.h"

namespace ts {
namespace {

// The merge of one (sequence, head) over its ns > 1 splits (body of decode_combine_kernel).
template <int HD>
__device__ __forceinline__ void combine_rows(const DecodeArgs &a, int head, int s, int ns, int tid) {
    constexpr int V4 = HD / 4, NG = 256 / V4;
    __shared__ float4 part[NG][V4];
    __shared__ float lpart[NG];
    __shared__ float wmax[4];
    const size_t hidx = (size_t)s * a.n_head + head;
    const float *ml = a.ws + (size_t)a.L.S * a.n_head * a.n_split * HD;
    const float *mm = ml + hidx * a.n_split;
    const float *ll = ml + (size_t)a.L.S * a.n_head * a.n_split + hidx * a.n_split;

    const int g = tid / V4, j = tid % V4;
    const float4 *o4 = reinterpret_cast<const float4 *>(a.ws + hidx * a.n_split * HD);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float lsum = 0.0f;
    if (ns <= 4 * NG) {
        // Up to 4 splits per row group: every load is issued at once (each thread reads all ns
        // maxima itself besides its own rows), so the merge is one memory round trip, with no
        // reduction round for the maximum.  (Batch 1 has more than NG splits per head.)
        constexpr int R = 4;
        float mv[R * NG];
#pragma unroll
        for (int i = 0; i < R * NG; i++) mv[i] = i < ns ? mm[i] : kMinit;
        float4 x[R];
        float lg[R], mg[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int i = g + r * NG;
            const bool mine = i < ns;
            x[r] = mine ? o4[(size_t)i * V4 + j] : make_float4(0.f, 0.f, 0.f, 0.f);
            lg[r] = mine ? ll[i] : 0.0f;
            mg[r] = mine ? mm[i] : kMinit;
        }
        float M = kMinit;
#pragma unroll
        for (int i = 0; i < R * NG; i++) M = fmaxf(M, mv[i]);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float e = g + r * NG < ns ? exp2f(mg[r] - M) : 0.0f;
            acc.x += e * x[r].x;
            acc.y += e * x[r].y;
            acc.z += e * x[r].z;
            acc.w += e * x[r].w;
            lsum += e * lg[r];
        }
    } else {
        float M = kMinit;
        for (int i = tid; i < ns; i += 256) M = fmaxf(M, mm[i]);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        if ((tid & 63) == 0) wmax[tid >> 6] = M;
        __syncthreads();
        M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
#pragma unroll 4
        for (int i = g; i < ns; i += NG) {
            const float e = exp2f(mm[i] - M);
            const float4 x = o4[(size_t)i * V4 + j];
            acc.x += e * x.x;
            acc.y += e * x.y;
            acc.z += e * x.z;
            acc.w += e * x.w;
            lsum += e * ll[i];
        }
    }
    part[g][j] = acc;
    if (j == 0) lpart[g] = lsum;
    __syncthreads();
    if (tid < V4 && 4 * tid < a.L.hdr) {
        float4 r = part[0][tid];
        float l = lpart[0];
#pragma unroll
        for (int k = 1; k < NG; k++) {
            const float4 x = part[k][tid];
            r.x += x.x;
            r.y += x.y;
            r.z += x.z;
            r.w += x.w;
            l += lpart[k];
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        float *o = a.out + hidx * a.L.hdr + 4 * tid;  // d_out rows of hdr floats
        o[0] = r.x * inv;
        o[1] = r.y * inv;
        o[2] = r.z * inv;
        o[3] = r.w * inv;
    }
}

// ---- G <= 16: QK^T on v_mfma_i32_16x16x64_i8 --------------------------------------------------
//
// QK^T runs in exact integer arithmetic, for up to 16 query heads per kv head in one, two or
// four halves of 4 heads (the description below is of one half; every other half has its own q
// operand and accumulators against the same K operand).  The B operand is K^T: column n of tile t is position
// 4n + t of the window, and lane 16 g + n supplies 16 dims of it as unsigned bytes -- the
// nibbles of two K words, even dims from (w & 0x0F0F0F0F), odd dims from (w >> 4) & 0x0F0F0F0F,
// 3 VALU ops per word.  The A operand holds q: row 4 h + c is base-128 digit c (c = 0 most
// significant) of head h's q, rotated and scaled to an integer of at most 2^27, so the 16 rows
// carry all 4 digits of all 4 heads.  The accumulators start at -8 * (sum of the row's digits),
// which takes the nibble bias out exactly, and the products are summed exactly in i32.  Output
// lane 16 h + n then holds the 4 digit sums of head h at position 4n + t; one f32 Horner step
// per digit gives the score (one rounding).  Each lane runs the softmax of its head at its 4
// positions; p * s_v goes through a per-wave LDS tile into the PV operand layout of the
// 16x16x32 f16 instruction (as above).

template <int HD>
struct Window8 {
    static constexpr int NKW = HD / 8, NTD = HD / 16;
    uint32_t kw[NKW];     // lane order q of k_word_idx: tile t, half m, word i at 2 (t HD/64 + m) + i
    uint32_t vw[2][NTD];  // V words, as Window
    floatx4 sk, sv;       // scales of positions base + 4n .. base + 4n + 3 (n = lane % 16)
};

// Buffer resources of one split for the integer kernel: K, V and both scale arrays (loads past
// the bound return zeros and touch no memory).
struct Streams4 {
    __amdgpu_buffer_rsrc_t k, v, sk, sv;
};

// Cache policy of the window loads: non-temporal.  Every byte is read exactly once per launch,
// and each instruction covers whole cache lines.
constexpr int kNT = 2;

// One window (64 positions from `base`, a multiple of 64): each K and V instruction reads one
// contiguous kilobyte (the cache's chunk order puts exactly this lane's operand words there);
// the scale instructions read the window's 256 bytes, every 16 bytes by the 4 lanes of a
// column.
template <int HD, int POL = kNT>
__device__ __forceinline__ void load_window8(Window8<HD> &w, const Streams4 &st, int base, int lane) {
    constexpr int NKW = HD / 8, NTD = HD / 16, ROWB = HD / 2;
#pragma unroll
    for (int j = 0; j < NKW / 4; j++) {
        const u32x4 t4 = __builtin_amdgcn_raw_buffer_load_b128(st.k, lane * 16 + j * 1024, base * ROWB, POL);
        w.kw[4 * j + 0] = t4[0]; w.kw[4 * j + 1] = t4[1]; w.kw[4 * j + 2] = t4[2]; w.kw[4 * j + 3] = t4[3];
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
        for (int q4 = 0; q4 < NTD / 4; q4++) {
            const u32x4 t4 = __builtin_amdgcn_raw_buffer_load_b128(st.v, lane * 16 + q4 * 1024 + b * (HD * 16), (base / 32) * (HD * 16), POL);
            w.vw[b][4 * q4 + 0] = t4[0]; w.vw[b][4 * q4 + 1] = t4[1];
            w.vw[b][4 * q4 + 2] = t4[2]; w.vw[b][4 * q4 + 3] = t4[3];
        }
    }
    const int so = (lane & 15) * 16;
    w.sk = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(st.sk, so, base * 4, POL));
    w.sv = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(st.sv, so, base * 4, POL));
}

template <int CTRL>
__device__ inline float dpp_any(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// Max / sum over the 16 lanes of a DPP row (every lane gets the result).
__device__ inline float row_max16(float v) {
    v = fmaxf(v, dpp_any<0xB1>(v));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp_any<0x4E>(v));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp_any<0x141>(v));  // row_half_mirror
    v = fmaxf(v, dpp_any<0x140>(v));  // row_mirror
    return v;
}
__device__ inline float row_sum16(float v) {
    v += dpp_any<0xB1>(v);
    v += dpp_any<0x4E>(v);
    v += dpp_any<0x141>(v);
    v += dpp_any<0x140>(v);
    return v;
}

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// Running state of one wave.  GH = 1 (G <= 4): O^T column n < 4 is head n from the high parts
// of p*s_v, 4 <= n < 8 head n - 4 from the low parts; GH = 2 (G <= 8): column n < 8 is head n
// from the high parts, 8 <= n < 16 head n - 8 from the low parts; GH = 4 (G <= 16): two sets
// of 16 columns, column n of set 0 head n from the high parts, of set 1 from the low parts.
// Lane 16 hg + n runs the softmax of heads hg + 4 hf (half hf): the exponent reference of each
// (uniform over the lane's row) and this lane's share of its softmax sum.
template <int GH>
constexpr int kPvSets = GH == 4 ? 2 : 1;
template <int HD, int GH>
struct WaveState8 {
    floatx4 o[kPvSets<GH>][HD / 16];
    float m[GH], l[GH];
};

// LDS slot of position `key` (0..63) of a window in the PV operand order: lane (n, g) of the
// 16x16x32 B operand reads slots 32b + 8g .. +7 = positions 32b + 16t + 4g + r at 2r + t.
__device__ inline int p_slot(int key) {
    return 32 * (key >> 5) + 8 * ((key >> 2) & 3) + 2 * (key & 3) + ((key >> 4) & 1);
}

// One window.  Half hf of the heads (4 hf .. 4 hf + 3) has its own q operand qa[hf] and bias:
// one i8 instruction per half and k-group, both on the same unpacked K operand.  pt: the wave's
// P tile, 8 GH columns.
template <int HD, bool SOFTCAP, int GH, bool SCORES = false>
__device__ __forceinline__ void process_window8(const Window8<HD> &w, WaveState8<HD, GH> &st,
                                                const i32x4 (&qa)[GH][HD / 64], const i32x4 (&bias)[GH],
                                                const float (&qinv)[GH], _Float16 (*pt)[64], int base, int end,
                                                int lane, const bool (&live)[GH], float softcap, const DeqConst &dc,
                                                float *scores = nullptr, int score_ld = 0, float inv_softcap = 0.0f) {
    constexpr int NTD = HD / 16, NM = HD / 64;
    const int n = lane & 15, hg = lane >> 4;
    // ---- S = Q K^T, exact -----------------------------------------------------------------
    i32x4 acc[GH][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
        for (int hf = 0; hf < GH; hf++) acc[hf][t] = bias[hf];
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const uint32_t w0 = w.kw[2 * (t * NM + m)], w1 = w.kw[2 * (t * NM + m) + 1];
            const i32x4 kb = {(int)(w0 & 0x0F0F0F0Fu), (int)((w0 >> 4) & 0x0F0F0F0Fu),
                              (int)(w1 & 0x0F0F0F0Fu), (int)((w1 >> 4) & 0x0F0F0F0Fu)};
#pragma unroll
            for (int hf = 0; hf < GH; hf++)
                acc[hf][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[hf][m], kb, acc[hf][t], 0, 0, 0);
        }
    }
    // ---- softmax of heads hg (+ 4 hf) at positions base + 4n + t --------------------------
    float x[GH][4], sv[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        sv[t] = base + 4 * n + t >= end ? 0.0f : w.sv[t];  // positions past the split's end
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            // digits 0..3 carry weights 2^21, 2^14, 2^7, 1; each digit sum is an exact integer
            // below 2^18, so the two pairs combine exactly in i32 (below 2^26) and the score
            // takes two conversions and one FMA.
            const int dhi = acc[hf][t][0] * 128 + acc[hf][t][1], dlo = acc[hf][t][2] * 128 + acc[hf][t][3];
            float v = fmaf((float)dhi, 16384.0f, (float)dlo);
            v *= qinv[hf] * w.sk[t];
            if constexpr (SOFTCAP && SCORES) v = cap<true>(v * (1.0f / kLog2e), softcap, inv_softcap);
            else if constexpr (SOFTCAP) v = tanhf(v * (1.0f / kLog2e) / softcap) * softcap * kLog2e;
            x[hf][t] = base + 4 * n + t >= end ? -INFINITY : v;
        }
    }
    if constexpr (SCORES) {
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            if (!live[hf]) continue;
            float *to = scores + (size_t)(hg + 4 * hf) * score_ld + base + 4 * n;
            if (base + 4 * n + 3 < end) {
                *reinterpret_cast<float4 *>(to) = make_float4(x[hf][0], x[hf][1], x[hf][2], x[hf][3]);
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
                    if (base + 4 * n + t < end) to[t] = x[hf][t];
            }
        }
    }
    // P = 2^(x - m) * s_v must stay <= 2^8 (f16 range for its two parts, with room).  The
    // reference m of a head moves only when some position of the window breaks that: a ballot
    // in the common case, row reductions only then (to m = max(x) + log2(max s_v), P <= 1).
    float p[GH][4], pv[GH][4];
    bool need = false;
#pragma unroll
    for (int hf = 0; hf < GH; hf++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            p[hf][t] = live[hf] ? fast_exp2(x[hf][t] - st.m[hf]) : 0.0f;
            pv[hf][t] = p[hf][t] * sv[t];
            need |= !(pv[hf][t] <= 256.0f);
        }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
        asm volatile("" ::: "memory");  // keep this a branch: the rescale is the rare case
        const float svl = __builtin_amdgcn_logf(row_max16(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]))));
        float al[GH];
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            const float xm = row_max16(fmaxf(fmaxf(x[hf][0], x[hf][1]), fmaxf(x[hf][2], x[hf][3])));
            const float mw = fminf(fmaxf(xm + svl, xm - 64.0f), xm + 64.0f);
            const float m_new = fmaxf(st.m[hf], mw);
            al[hf] = fast_exp2(st.m[hf] - m_new);
            st.l[hf] *= al[hf];
            st.m[hf] = m_new;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                p[hf][t] = live[hf] ? fast_exp2(x[hf][t] - st.m[hf]) : 0.0f;
                pv[hf][t] = p[hf][t] * sv[t];
            }
        }
        // the O^T columns of head c take the factor of its row: head c of half hf is row c % 4
        // of al[hf] (lane 16 (c % 4))
        const int c = GH == 1 ? (lane & 3) : GH == 2 ? (lane & 7) : (lane & 15);
        float f = 1.0f;
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            const float f0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al[hf]), 0));
            const float f1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al[hf]), 16));
            const float f2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al[hf]), 32));
            const float f3 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al[hf]), 48));
            const int cc = c & 3;
            if ((c >> 2) == hf) f = cc == 0 ? f0 : cc == 1 ? f1 : cc == 2 ? f2 : f3;
        }
#pragma unroll
        for (int ps = 0; ps < kPvSets<GH>; ps++)
#pragma unroll
            for (int td = 0; td < NTD; td++) st.o[ps][td] *= f;
    }
#pragma unroll
    for (int hf = 0; hf < GH; hf++) st.l[hf] += (p[hf][0] + p[hf][1]) + (p[hf][2] + p[hf][3]);
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int slot = p_slot(4 * n + t);
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            const float hi = split_hi(pv[hf][t]);
            pt[4 * hf + hg][slot] = (_Float16)hi;
            pt[4 * GH + 4 * hf + hg][slot] = (_Float16)(pv[hf][t] - hi);
        }
    }
    // ---- O^T += V^T P^T (the wave's own LDS writes are ordered before its reads) -------------
    const int g = lane >> 4;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        // GH = 1: columns 8..15 read real p values; their outputs are never used
        half8 pb[kPvSets<GH>];
#pragma unroll
        for (int ps = 0; ps < kPvSets<GH>; ps++)
            pb[ps] = *reinterpret_cast<const half8 *>(&pt[GH == 1 ? (n & 7) : 16 * ps + n][32 * b + 8 * g]);
        // every word of the block dequantized into its own registers first, so the conversions
        // of later words overlap the matrix instructions of earlier ones
        half8 va[NTD];
#pragma unroll
        for (int td = 0; td < NTD; td++) va[td] = dequant8(w.vw[b][td], dc);
#pragma unroll
        for (int ps = 0; ps < kPvSets<GH>; ps++)
#pragma unroll
            for (int td = 0; td < NTD; td++)
                st.o[ps][td] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[td], pb[ps], st.o[ps][td], 0, 0, 0);
    }
}

// NW waves per workgroup, D windows in registers per wave (D - 1 in flight while one is
// computed).  The plan places one workgroup per CU (NW = 4: one wave per SIMD; NW = 8 for
// 64-dim rows: two).
// PAD: the caller's head dim hdr is below the stored HD (rows of q, new K/V and the output are
// hdr floats; the stored dims past them hold code 8 = 0, so the integer QK^T and PV run
// unchanged over the whole stored row).
// GH: halves of 4 query heads per wave (1: G <= 4, 2: G <= 8, 4: G <= 16).  HG: head groups of
// the workgroup: with HG = 2, waves 0 .. NW/2 - 1 take query heads 0..7 and the others heads
// 8..15, both groups over the same windows in the same order (the second read of a window
// comes from L2, so cached loads), each with NW/2 waves.
template <int HD, bool SOFTCAP, bool NORM, bool PAD, int NW, int D, int GH, int HG = 1, bool SCORES = false>
__global__ __launch_bounds__(64 * NW, NW / 4) void decode_split4_kernel(DecodeArgs a) {
    constexpr int NTD = HD / 16;
    constexpr int NM = HD / 64;  // i8 instructions per 16-position tile
    constexpr int OST = HD + 4;  // 16-byte rows of the merge area
    const KvLayerView &L = a.L;
    const int hdr = PAD ? L.hdr : HD;
    const float *const QN = NORM ? L.qn : nullptr;  // QK norm of q (compiled out when off)
    // grid (kv head, sequence, split): every sequence's split 0 is dispatched before any
    // split 1, so the splits that wait for a free CU are the last ones of the longest
    // sequences (config 4: 1.42 vs 1.45 ms per step against the split-fastest order)
    const int split = blockIdx.z, h = blockIdx.x, s = blockIdx.y;
    int qpos, qrot;  // the query's slot and rotation position
    token_pos(a, s, qpos, qrot);
    // a captured launch replayed past the cache's capacity (the host checks lengths only when a
    // call is made): no work, nothing written
    if (qpos >= L.P) return;
    const int n_ctx = qpos + 1;
    const int start = split * a.chunk;
    if (start >= n_ctx) return;
    const int n_split_s = min((n_ctx + a.chunk - 1) / a.chunk, a.n_split);
    const bool fused = a.k_new != nullptr && split == n_split_s - 1;
    // the last split runs to the end, also past chunk * n_split (a launch captured for shorter
    // contexts stays correct, only less balanced)
    const int end = fused ? qpos : (split == n_split_s - 1 ? n_ctx : start + a.chunk);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.G;
    const DeqConst dc;

    // per-wave p*s_v tiles, [column][slot]; and the merge area, apart from them so that a wave
    // writes its share of the merge as soon as its windows are done
    __shared__ _Float16 pts[NW][8 * GH][64];
    __shared__ __align__(16) float mo[NW][8 * GH * OST];  // O^T columns, OST floats apart
    __shared__ float mm_[NW][4 * GH], ml_[NW][4 * GH];
    __shared__ __align__(16) float kd[HD], vd[HD];
    __shared__ float xnew[4 * GH * HG < 8 ? 8 : 4 * GH * HG];
    __shared__ float lse_s[SCORES ? 16 : 1];
    __shared__ int32_t qsum[NW][GH][16];  // per wave and half: digit sums of the 16 q rows
    __shared__ float qinv_s[NW][GH][4];   // per wave and half: 2^-e of each head's q scale

    const size_t row = (size_t)s * L.H + h;
    constexpr int ROWB = HD / 2;
    Streams4 str;
    // K and the scales are bounded at the window: a window's K chunks mix its rows, and a
    // scale load covers 4 positions
    const uint32_t wend = (uint32_t)((end + 63) & ~63);
    str.k = make_rsrc(L.kp + row * L.P * ROWB, wend * ROWB);
    str.v = make_rsrc(L.vp + row * (L.P / 32) * (HD * 16), (uint32_t)((end + 31) / 32) * (HD * 16));
    str.sk = make_rsrc(L.ks + row * L.P, wend * 4);
    str.sv = make_rsrc(L.vs + row * L.P, wend * 4);

    // This wave's windows: claims j = wave, wave + NW, ... below nwin, taken in rotated order
    // starting at a per-workgroup offset, so that the workgroups streaming at the same time
    // read different regions of their streams (spread over the HBM channels).  Claim j reads
    // window (j + R) mod nwin.  The appending wave starts ~3 us late, so it keeps all but its
    // last kApp claims, which go round robin to the other waves after their own: the
    // assignment stays fixed (outputs are bit-reproducible) and the waves end together.
    // (Without the hand-over the appending wave ended ~2 us after the others: config 3
    // 1.880 vs 1.855 ms per step, measured with claims through an LDS counter.)  Window
    // indices past the wave's count load from past the bound (zeros, no memory traffic).
    // (per head group: NWG waves, wave wl of group hgp; only the appending wave's group hands
    // windows over)
    constexpr int NWG = NW / HG;
    const int hgp = __builtin_amdgcn_readfirstlane(wave / NWG), wl = wave - NWG * hgp;
    const int nwin = (end - start + 63) >> 6;
    const int own = wl < nwin ? (nwin - wl + NWG - 1) / NWG : 0;
    const int lastc = NWG - 1 < nwin ? (nwin - (NWG - 1) + NWG - 1) / NWG : 0;  // the last wave's claims
    const int kApp = fused && hgp == HG - 1 ? min(3, lastc / 3) : 0;
    const int keep = lastc - kApp;  // claims the last wave keeps
    const int extra = wl < NWG - 1 ? (kApp - wl + NWG - 2) / (NWG - 1) : 0;
    const int cnt = wl < NWG - 1 ? own + extra : keep;
    // (s 13 + h 5 + split 7: the workgroups on one XCD -- the same kv head for one split --
    // start at distinct windows; measured against (row 37 + split 11), whose offsets repeat
    // every 4 sequences of a head: config 3 1.798 vs 1.834 ms per step)
    const int R = nwin ? (int)((unsigned)(NWG * (s * 13 + h * 5 + split * 7)) % (unsigned)nwin) : 0;
    const int oob = start + 64 * nwin;
    auto win_base = [&](int i) {
        if (i >= cnt) return oob;
        const int j = i < own ? NWG * i + wl : NWG * (keep + (NWG - 1) * (i - own) + wl) + NWG - 1;
        int r = j + R;
        r = r >= nwin ? r - nwin : r;
        return start + 64 * r;
    };
    Window8<HD> w[D];
    // this wave's query heads: Gg of them from head hgb of the sequence (HG = 2: up to 8 a group)
    const int Gg = HG == 1 ? G : max(0, min(8, G - 8 * hgp));
    const int hgb = h * G + (HG == 1 ? 0 : 8 * hgp);

    // q operand: lane 16 g + n holds row n = 4 hh + c (digit c of head hh) for k-group g, i.e.
    // dims 64 m + 16 g .. + 15 of instruction m, bytes [even dims of word 8m + 2g, its odd
    // dims, even dims of word 8m + 2g + 1, its odd dims] like the K operand.  The raw q loads
    // go out before the windows' prefetch: loads complete in order, so consuming q then does
    // not wait for the windows.
    i32x4 qa[GH][NM], bias[GH];
    float qinv[GH];
    const bool appender = fused && wave == NW - 1;
    AppendIn<HD> ain;
    float2 qp[4 * GH * HG][AppendIn<HD>::PPL];
    {
        // half hf: lane 16 g + n holds digit dg of head hh + 4 hf
        const int n = lane & 15, g = lane >> 4, hh = n >> 2, dg = n & 3;
        bool hl[GH];
        float qx[GH][NM][16], nwv[NM][16];
        float2 qcs[NM][8];
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            hl[hf] = hh + 4 * hf < Gg;
            const float *qrow = a.q + ((size_t)s * a.n_head + hgb + (hl[hf] ? hh + 4 * hf : 0)) * hdr;
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const int d0 = 64 * m + 16 * g;
#pragma unroll
                for (int e4 = 0; e4 < 4; e4++) {
                    const bool in = d0 + 4 * e4 < hdr;  // stored dims past the row are 0
                    const float4 v4 = keep4(in, *reinterpret_cast<const float4 *>(qrow + (in ? d0 + 4 * e4 : 0)));
                    qx[hf][m][4 * e4] = v4.x; qx[hf][m][4 * e4 + 1] = v4.y;
                    qx[hf][m][4 * e4 + 2] = v4.z; qx[hf][m][4 * e4 + 3] = v4.w;
                }
            }
        }
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const int d0 = 64 * m + 16 * g;
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
                const bool in = d0 + 4 * e4 < hdr;
                if (QN) {
                    const float4 n4 = *reinterpret_cast<const float4 *>(QN + (in ? d0 + 4 * e4 : 0));  // (only
                    // multiplies dims that are zero past the row)
                    nwv[m][4 * e4] = n4.x; nwv[m][4 * e4 + 1] = n4.y; nwv[m][4 * e4 + 2] = n4.z; nwv[m][4 * e4 + 3] = n4.w;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int pair = d0 / 2 + i;
                qcs[m][i] = pair < a.rope_pairs
                                ? *reinterpret_cast<const float2 *>(a.rope + ((size_t)qrot * a.rope_pairs + pair) * 2)
                                : make_float2(1.0f, 0.0f);
            }
        }
        // QK norm scale of this lane's head in each half (all heads' scales, then a select)
        float ns[GH];
#pragma unroll
        for (int hf = 0; hf < GH; hf++) ns[hf] = 1.0f;
        if (QN) {
            float nall[4 * GH];
            q_norm_scales_wave<HD, 4 * GH>(a.q + ((size_t)s * a.n_head + hgb) * hdr, Gg, L.norm_eps, hdr, nall);
#pragma unroll
            for (int hf = 0; hf < GH; hf++)
#pragma unroll
                for (int c = 0; c < 4; c++) ns[hf] = hh == c ? nall[4 * hf + c] : ns[hf];
        }
        // The appending wave (the last: it has the fewest windows) quantizes the new token and
        // scores it against every head before its windows; the others start at once.  Its
        // loads go out with q's.  kd, vd and xnew are read after the barrier that opens the
        // merge.
        if (appender) {
            append_load<HD, NORM>(a, s, h, qpos, qrot, lane, ain, hdr);
            load_q_pairs<HD, 4 * GH * HG>(a, s, h * G, G, lane, qp, hdr);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < D - 1; d++) load_window8<HD, HG == 1 ? kNT : 0>(w[d], str, win_base(d), lane);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
        // rotated q times log2(e)/sqrt(hd) (rope.rs:186-196 after the optional QK norm)
        float qm = 0.0f;
#pragma unroll
        for (int m = 0; m < NM; m++) {
#pragma clang fp contract(off)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float x0 = qx[hf][m][2 * i], x1 = qx[hf][m][2 * i + 1];
                if (QN) {
                    x0 = qk_norm_apply(x0, ns[hf], nwv[m][2 * i]);
                    x1 = qk_norm_apply(x1, ns[hf], nwv[m][2 * i + 1]);
                }
                if ((64 * m + 16 * g) / 2 + i < a.rope_pairs) rope_rotate(x0, x1, qcs[m][i]);
                qx[hf][m][2 * i] = x0 * (a.inv_sqrt_hd * kLog2e);
                qx[hf][m][2 * i + 1] = x1 * (a.inv_sqrt_hd * kLog2e);
                qm = fmaxf(qm, fmaxf(fabsf(qx[hf][m][2 * i]), fabsf(qx[hf][m][2 * i + 1])));
            }
        }
        // head hh's integer scale 2^e: max |q| 2^e in [2^26, 2^27), so every digit fits int8
        qm = group_max(qm);
        int e = 0;
        if (qm > 0.0f && qm < 3.0e38f) e = 26 - min(max(ilogbf(qm), -100), 100);
        const float sc = ldexpf(1.0f, e);
        // digits: Q = d0 2^21 + d1 2^14 + d2 2^7 + d3, d1..d3 in [-64, 63], |d0| <= 64.  With
        // Q' = Q + 64 (2^21 + 2^14 + 2^7 + 1) > 0, D_c = d_c + 64 are the base-128 digits of Q'
        // (D_0 = Q' >> 21 <= 128), so this lane's digit is one shift and mask away.
        const int sh = 7 * (3 - dg);
        const uint32_t msk = dg == 0 ? 0xFFu : 0x7Fu;
        uint32_t dsum_raw = 0;
#pragma unroll
        for (int m = 0; m < NM; m++) {
            uint32_t reg[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int el = 0; el < 16; el++) {
                const int Q = hl[hf] ? (int)rintf(qx[hf][m][el] * sc) : 0;
                const uint32_t dig = ((uint32_t)(Q + 135274560) >> sh) & msk;
                dsum_raw += dig;
                // element el = dim 64 m + 16 g + el: word 8m + 2g + el / 8, parity el % 2 selects
                // the even (reg 0 / 2) or odd (reg 1 / 3) register, byte (el % 8) / 2
                const int rr = 2 * (el >> 3) + (el & 1), by = (el & 7) >> 1;
                reg[rr] |= ((dig + 192u) & 0xFFu) << (8 * by);  // the byte of D_c - 64
            }
            qa[hf][m] = (i32x4){(int)reg[0], (int)reg[1], (int)reg[2], (int)reg[3]};
        }
        int dsum = (int)dsum_raw - 64 * 16 * NM;
        // bias of accumulator (head hg, digit r): -8 * (digit sum of row 4 hg + r)
        dsum += __shfl_xor(dsum, 16, 64);
        dsum += __shfl_xor(dsum, 32, 64);
        if (g == 0) qsum[wave][hf][n] = dsum;
        if (g == 0 && dg == 0) qinv_s[wave][hf][hh] = ldexpf(1.0f, -e);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's LDS writes are done
        __builtin_amdgcn_wave_barrier();
        const int hg = lane >> 4;
#pragma unroll
        for (int hf = 0; hf < GH; hf++) {
            bias[hf] = (i32x4){-8 * qsum[wave][hf][4 * hg], -8 * qsum[wave][hf][4 * hg + 1],
                               -8 * qsum[wave][hf][4 * hg + 2], -8 * qsum[wave][hf][4 * hg + 3]};
            qinv[hf] = qinv_s[wave][hf][hg];
        }
    }
    if (appender) {
        append_store<HD, NORM>(a, s, h, qpos, lane, ain, kd, vd, hdr);
        new_token_scores<HD, SOFTCAP, NORM, 4 * GH * HG>(a, s, h * G, G, lane, qp, ain.cs, kd, xnew, hdr);
    }

    WaveState8<HD, GH> st;
#pragma unroll
    for (int ps = 0; ps < kPvSets<GH>; ps++)
#pragma unroll
        for (int td = 0; td < NTD; td++) st.o[ps][td] = (floatx4)0.0f;
    bool live[GH];
#pragma unroll
    for (int hf = 0; hf < GH; hf++) {
        st.m[hf] = kMinit;
        st.l[hf] = 0.0f;
        live[hf] = (lane >> 4) + 4 * hf < Gg;
    }
    _Float16 (*pt)[64] = pts[wave];
    float *const scores = SCORES ? a.scores + ((size_t)s * a.n_head + hgb) * L.P : nullptr;

    int it = 0;
    if (cnt > 0) {
        while (true) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                load_window8<HD, HG == 1 ? kNT : 0>(w[(d + D - 1) % D], str, win_base(it + D - 1), lane);
                // keep the prefetch here: the scheduler would otherwise sink it below the use.
                // (Refilling a slot right after its window is processed instead measured
                // slower: config 3 1.871 vs 1.848 ms per step, config 4 1.63 vs 1.46.)
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                // (one form for every window, the tail mask included: a branch between a masked
                // and an unmasked copy made the compiler shuffle the accumulators at the join,
                // ~30 moves per window; config 4 1.396 vs 1.408 ms per step)
                process_window8<HD, SOFTCAP, GH, SCORES>(w[d], st, qa, bias, qinv, pt, win_base(it), end, lane, live, a.softcap, dc, scores, L.P, a.inv_softcap);
                if (++it >= cnt) goto windows_done;
            }
        }
    }
windows_done:

    // ---- merge the waves through LDS ------------------------------------------------------------
    // Each wave writes its O^T columns (16-byte stores: lane (n, g) holds dims 16 td + 4 g ..
    // + 3 of column n), its m and l; one barrier; then one float4 of dims per thread.
    // (Merge area shared with the P tiles, a barrier before the writes, scalar stores and one
    // dim per thread: ~1.4 us from the last wave's loop end to the output.)
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int hf = 0; hf < GH; hf++) {
        const float l_run = row_sum16(st.l[hf]);
        if (n == 0) {
            mm_[wave][4 * hf + g] = st.m[hf];
            ml_[wave][4 * hf + g] = l_run;
        }
    }
#pragma unroll
    for (int ps = 0; ps < kPvSets<GH>; ps++)
        if (16 * ps + n < 8 * GH) {
#pragma unroll
            for (int td = 0; td < NTD; td++)
                *reinterpret_cast<floatx4 *>(&mo[wave][(16 * ps + n) * OST + 16 * td + 4 * g]) = st.o[ps][td];
        }
    __syncthreads();

    constexpr int V4 = HD / 4;
    for (int idx = tid; idx < G * V4; idx += 64 * NW) {
        const int hh = idx / V4, d = 4 * (idx % V4);
        // head hh is head lh of group grp, held by that group's NWG waves from wave wb
        const int grp = HG == 1 ? 0 : hh >> 3, lh = hh - 8 * grp, wb = NWG * grp;
        float M = kMinit;
#pragma unroll
        for (int w = 0; w < NWG; w++) M = fmaxf(M, mm_[wb + w][lh]);
        if (fused) M = fmaxf(M, xnew[hh]);
        floatx4 acc = (floatx4)0.0f;
        float lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < NWG; w++) {
            const float e = exp2f(mm_[wb + w][lh] - M);
            const floatx4 hi = *reinterpret_cast<const floatx4 *>(&mo[wb + w][lh * OST + d]);
            const floatx4 lo = *reinterpret_cast<const floatx4 *>(&mo[wb + w][(lh + 4 * GH) * OST + d]);
            acc += e * (hi + lo);
            lsum += e * ml_[wb + w][lh];
        }
        if (fused) {
            const float e = exp2f(xnew[hh] - M);
            acc += e * *reinterpret_cast<const floatx4 *>(&vd[d]);
            lsum += e;
        }
        const size_t head = (size_t)s * a.n_head + h * G + hh;
        if constexpr (SCORES) {
            if (d == 0) {
                if (fused) a.scores[head * L.P + qpos] = xnew[hh];
                if (n_split_s == 1 && !a.w) store_stats(a, head, split, HD, M, lsum);
                lse_s[hh] = M + __log2f(lsum);
            }
        }
        if (n_split_s == 1) {
            // hdr is a multiple of 8: a float4 of dims lies wholly inside or outside the row
            const float inv = lsum > 0.0f ? 1.0f / lsum : 0.0f;
            if (d < hdr) {
                const floatx4 r = lsum > 0.0f ? acc * inv : (floatx4)0.0f;
                *reinterpret_cast<float4 *>(a.out + head * hdr + d) = make_float4(r[0], r[1], r[2], r[3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) store_partial(a, head, split, HD, d + k, acc[k], M, lsum);
        }
    }
    if constexpr (SCORES) {
        if (a.w) {  // (every slot of the stream is this workgroup's)
            __syncthreads();
            add_weights<4 * GH * HG, 64 * NW>(a, row, (size_t)s * a.n_head + h * G, G, n_ctx, lse_s, tid);
        }
    }
}

// The integer kernel's static LDS (the arrays it declares), for the dynamic reservation below.
template <int HD, int NW, int GH, int HG>
constexpr size_t split4_static_lds() {
    return (size_t)NW * 8 * GH * 64 * 2          // pts
           + (size_t)NW * 8 * GH * (HD + 4) * 4  // mo
           + (size_t)2 * NW * 4 * GH * 4         // mm_, ml_
           + (size_t)2 * HD * 4 + (4 * GH * HG < 8 ? 8 : 4 * GH * HG) * 4  // kd, vd, xnew
           + (size_t)NW * GH * 16 * 4 + (size_t)NW * GH * 4 * 4;  // qsum, qinv_s
}

// One integer-kernel launch.  The kernel fits two workgroups per CU by registers, but the plan
// wants one per CU: an unused dynamic LDS reservation that takes the workgroup to 84 KB (more
// than half of a CU's 160 KB, and at most all of it) makes the dispatcher place busy workgroups
// on distinct CUs, also when the grid holds idle ones (splits past a short sequence's end)
// that exit at once.
template <int HD, bool SC, bool NM, bool PAD, int NW, int GH, int HG = 1, bool SCORES = false>
void launch_split4(const DecodeArgs &a, int n_split, hipStream_t st) {
    constexpr size_t kOne = 84 * 1024, own = split4_static_lds<HD, NW, GH, HG>();
    static_assert(own <= 160 * 1024, "integer kernel LDS");
    constexpr size_t lds = own >= kOne ? 0 : kOne - own;
    decode_split4_kernel<HD, SC, NM, PAD, NW, 2, GH, HG, SCORES><<<dim3(a.L.H, a.L.S, n_split), 64 * NW, lds, st>>>(a);
}

// 64-dim rows carry half the bytes per position for the same per-position softmax work: they
// run 8 waves (two per SIMD), so that one wave's softmax overlaps the other's loads.  Config-3
// shape with 64-dim rows: 1.170 vs 1.378 ms per step at 8 query heads per kv head, 1.017 vs
// 1.030 at 4; ragged config 4: 0.837 vs 0.886.  (With 128-dim rows and two halves of heads 8
// waves measured slower: 1.970 vs 1.888.)
// With the scores (SCORES) 128-dim rows run 8 waves too, one storing while the other loads: 32 sequences of 4096-8192
// slots 56 us, with 4 waves 60; 8 of 1001-16003 26.6 and 27.5.
template <int HD, bool SC, bool NM, bool SCORES = false>
void launch_integer(const DecodeArgs &a, int n_split, bool pad, int Gt, hipStream_t st) {
    constexpr int NW = HD == 64 || (SCORES && HD == 128) ? 8 : 4;
    if constexpr (HD <= 128) {
        // More than 8 query heads per kv head (the plan allows them up to 128-dim rows).  On
        // 64-dim rows: two head groups of 4 waves, two halves each (config-3 shape with 128 q
        // heads 1.955 vs 2.199 ms per step); on 128-dim rows: four halves in one wave per SIMD
        // (2.86 vs 3.39 ms with head groups, whose second read of each window does not all come
        // from L2).
        if (Gt > 8) {
            if constexpr (HD == 64) {
                if (pad) launch_split4<HD, SC, NM, true, 8, 2, 2, SCORES>(a, n_split, st);
                else launch_split4<HD, SC, NM, false, 8, 2, 2, SCORES>(a, n_split, st);
            } else {
                if (pad) launch_split4<HD, SC, NM, true, 4, 4, 1, SCORES>(a, n_split, st);
                else launch_split4<HD, SC, NM, false, 4, 4, 1, SCORES>(a, n_split, st);
            }
            return;
        }
    }
    if (Gt > 4) {
        if (pad) launch_split4<HD, SC, NM, true, NW, 2, 1, SCORES>(a, n_split, st);
        else launch_split4<HD, SC, NM, false, NW, 2, 1, SCORES>(a, n_split, st);
    } else {
        if (pad) launch_split4<HD, SC, NM, true, NW, 1, 1, SCORES>(a, n_split, st);
        else launch_split4<HD, SC, NM, false, NW, 1, 1, SCORES>(a, n_split, st);
    }
}

}  // namespace
}  // namespace ts
