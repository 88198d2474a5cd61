// ts_prompt.hip -- causal attention over packed prompts for gfx950: per sequence
//   o_t = sum_{j <= t} softmax_j(cap(q_t k_j / sqrt(hd))) v_j,   cap(x) = softcap tanh(x / softcap),
// in one pass over the keys with the running maximum and sum of the softmax.
//
// * The (token, head) pairs that share one kv head form the columns of the matrix products, as in
//   chunked prefill: column c is token c / G, head c % G, so that a tile of K and V serves all G
//   heads, and a short sequence still fills its columns.
// * A workgroup of 4 waves owns 128 columns (32 a wave) and walks the keys up to its last token in
//   tiles that all waves share through LDS.
// * S^T = K Q^T leaves each lane with scores of one column; the keys it holds are those it supplies
//   to O^T = V^T P^T, so P stays in registers.  V^T comes out of the row-major tile through
//   transposing LDS reads.
// * f16 and bf16 rows go into the matrix cores as they are; P is rounded once to the same type.
//   f32 rows are split by a first kernel into two f16 planes (hi + lo, 22 bits) with a power of two
//   per row that takes its largest element to [2^13, 2^14); products hi hi + hi lo + lo hi.
// Scores, maxima, sums and outputs are f32 until the output is rounded once.
#include "ts_prompt.h"

#include "ts_mfma.h"

namespace ts {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));

constexpr int kPromptNW = 4;
constexpr int kPromptCols = 32 * kPromptNW;

struct PromptArgs {
    const void *q, *k, *v;
    void *out;
    int64_t qs, ks, vs, os;
    // f32: planes [rows][n_kv][2 hdp] of K and V, per row (of row0 on) and head the exponents
    const _Float16 *kp, *vp;
    const float *ke, *ve;
    int64_t row0;
    int G, H, hd;
    float scale;  // 1 / sqrt(hd), times log2(e) without softcap
    float softcap;
    PackTable t;
};

__device__ inline floatx16 mfma(f16x8 a, f16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

template <class T>
struct Vec8;
template <>
struct Vec8<_Float16> { using type = f16x8; };
template <>
struct Vec8<__bf16> { using type = bf16x8; };

__device__ inline float both_max(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float both_sum(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Slot of 16-byte chunk c in row r of a tile: K rows are read 8 and more at a time at one chunk, V
// rows 4 at a time over 64 bytes; the XOR puts those on distinct banks.
template <int CPR>
__device__ inline int kslot(int r, int c) { return c ^ (r & (CPR < 16 ? CPR - 1 : 15)); }
template <int CPR>
__device__ inline int vslot(int r, int c) { return c ^ (CPR < 16 ? (r & 1) << 2 : (r & 3) << 2); }

// The 8 keys of one lane of a 16-key step, of one dim (lane % 32 of tile db): rows 4h .. and 8 + 4h ..
// of the step.  Each group of 16 lanes reads 4 rows x 16 dims and gets them transposed.
template <class T, int CPR>
__device__ inline typename Vec8<T>::type v_operand(const u32x4 *tile, int row0, int chunk0, int lane) {
    const int i = lane & 15, r = row0 + 4 * (lane >> 5) + (i >> 2), c = chunk0 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    typedef __attribute__((address_space(3))) short4v *lds4;
    auto at = [&](int row) {
        return (lds4)(reinterpret_cast<const short4v *>(tile + row * CPR + vslot<CPR>(row, c)) + (i & 1));
    };
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(r)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(r + 8));
    const short8v s = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(typename Vec8<T>::type, s);
}

// Whether any of 8 elements is infinite or NaN.
template <class V>
__device__ inline bool any_bad(V v, bool f16) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    const uint32_t m = f16 ? 0x7C00u : 0x7F80u;
    auto bad = [&](uint32_t x) { return (x & m) == m || ((x >> 16) & m) == m; };
    return bad(w.x) || bad(w.y) || bad(w.z) || bad(w.w);
}
// v with every element that is not finite replaced: by 0 (part 0), or all others by 0 and those by 1
// where they are +inf or NaN (part 1), -inf or NaN (part 2).
template <class T>
__device__ inline typename Vec8<T>::type bad_part(typename Vec8<T>::type v, int part) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float x = (float)v[e];
        const bool bad = !(fabsf(x) < INFINITY);
        const bool hit = part == 1 ? bad && !(x < 0.0f) : bad && !(x > 0.0f);
        v[e] = part == 0 ? (bad ? (T)0.0f : v[e]) : hit ? (T)1.0f : (T)0.0f;
    }
    return v;
}

// T: the matrix cores' type; O: the rows' type (float with two planes); HD: head dims, padded; NP:
// planes; KT: keys per tile.
template <class T, class O, int HD, int NP, int KT, bool SOFTCAP>
__global__ __launch_bounds__(64 * kPromptNW, HD * NP > 128 ? 1 : 2) void prompt_kernel(PromptArgs a) {
    using V8 = typename Vec8<T>::type;
    constexpr int CPR = NP * HD / 8;  // 16-byte chunks of a tile's row
    constexpr int NKS = HD / 16, NDB = HD / 32, NKB = KT / 32;
    constexpr int NT = 64 * kPromptNW, NPC = KT * CPR / NT;  // pieces of a tile per thread
    constexpr bool F16 = sizeof(T) == 2 && __is_same(T, _Float16);
    static_assert(KT * CPR % NT == 0 && NPC > 0, "a tile's pieces spread evenly");
    extern __shared__ __align__(16) unsigned char pr_smem[];
    u32x4 *const kt = reinterpret_cast<u32x4 *>(pr_smem);  // [2][KT][CPR]
    u32x4 *const vt = kt + 2 * KT * CPR;
    float *const se = reinterpret_cast<float *>(vt + 2 * KT * CPR);  // two planes: [2][2][KT] K and V exponents

    const int item = blockIdx.x / a.H, h = blockIdx.x - item * a.H;
    const int i = pack_find(a.t, item);
    const int row0 = a.t.tok[i], n = a.t.tok[i + 1] - row0;
    const int G = a.G, n_cols = n * G;
    const int cblk = a.t.item[i + 1] - 1 - item;  // later tokens, the longer walks, first
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, hf = lane >> 5;
    const int c_blk = cblk * kPromptCols, c_wave = c_blk + 32 * wave;
    const int c = c_wave + j;
    const bool live = c < n_cols;
    const int cc = live ? c : n_cols - 1;
    const int tok = cc / G;
    const int head = h * G + cc - tok * G;
    const int hd = a.hd;
    const int n_chunk = hd / 8;

    // Tiles through registers into LDS.
    u32x4 pk[NPC], pv[NPC];
    float pe = 0.0f;
    auto fetch = [&](int base) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NPC; p++) {
            const int idx = tid + NT * p, r = idx / CPR, ch = idx % CPR;
            const int64_t row = row0 + min(base + r, n - 1);  // (keys past the end are masked)
            if constexpr (NP == 1) {
                // (chunks past the row repeat its last: q is 0 there, and those outputs are dropped)
                const int cl = min(ch, n_chunk - 1);
                pk[p] = *reinterpret_cast<const u32x4 *>(static_cast<const T *>(a.k) + row * a.ks + (int64_t)h * hd + 8 * cl);
                pv[p] = *reinterpret_cast<const u32x4 *>(static_cast<const T *>(a.v) + row * a.vs + (int64_t)h * hd + 8 * cl);
            } else {
                const int64_t at = ((row - a.row0) * a.H + h) * (NP * HD) + 8 * ch;
                pk[p] = *reinterpret_cast<const u32x4 *>(a.kp + at);
                pv[p] = *reinterpret_cast<const u32x4 *>(a.vp + at);
            }
        }
        if constexpr (NP == 2)
            if (tid < 2 * KT) {
                const int64_t at = (row0 - a.row0 + min(base + tid % KT, n - 1)) * a.H + h;
                pe = tid < KT ? a.ke[at] : a.ve[at];
            }
    };
    auto stage = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NPC; p++) {
            const int idx = tid + NT * p, r = idx / CPR, ch = idx % CPR;
            kt[(buf * KT + r) * CPR + kslot<CPR>(r, ch)] = pk[p];
            vt[(buf * KT + r) * CPR + vslot<CPR>(r, ch)] = pv[p];
        }
        if constexpr (NP == 2)
            if (tid < 2 * KT) se[buf * 2 * KT + tid] = pe;
    };
    fetch(0);

    // q of this lane's column: k-step t holds dims 16 t + 8 hf ..
    V8 qh[NKS], ql[NP == 2 ? NKS : 1];
    float qscale = a.scale;
    if constexpr (NP == 1) {
        const T *qrow = static_cast<const T *>(a.q) + (row0 + tok) * a.qs + (int64_t)head * hd;
#pragma unroll
        for (int t = 0; t < NKS; t++) {
            const bool in = 2 * t + hf < n_chunk;
            const V8 x = *reinterpret_cast<const V8 *>(qrow + (in ? 8 * (2 * t + hf) : 0));
#pragma unroll
            for (int e = 0; e < 8; e++) qh[t][e] = in ? x[e] : (T)0.0f;
        }
    } else {
        const float *qrow = static_cast<const float *>(a.q) + (row0 + tok) * a.qs + (int64_t)head * hd;
        float x[NKS][8], m = 0.0f;
#pragma unroll
        for (int t = 0; t < NKS; t++) {
            const bool in = 2 * t + hf < n_chunk;
            load8(qrow + (in ? 8 * (2 * t + hf) : 0), x[t]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[t][e] = in ? x[t][e] : 0.0f;
                m = fmaxf(m, fabsf(x[t][e]));
            }
        }
        float s, inv;
        q_scale(both_max(m), s, inv);
        qscale = a.scale * inv;
#pragma unroll
        for (int t = 0; t < NKS; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = opaque(x[t][e] * s);
                const _Float16 hi = (_Float16)v;
                qh[t][e] = (T)hi;
                ql[t][e] = (T)(v - (float)hi);
            }
    }

    const int qpos = live ? tok : -1;
    const int qmin_w = c_wave / G;
    const int qmax_w = c_wave < n_cols ? (min(c_wave + 32, n_cols) - 1) / G : -1;
    const int n_key = (min(c_blk + kPromptCols, n_cols) - 1) / G + 1;
    const int n_tile = (n_key + KT - 1) / KT;

    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) o[db] = (floatx16)0.0f;
    float m_run = -3.4e38f, l_run = 0.0f;  // (below every finite score: the first tile sets it)
    // P is held up to 2^(8 + kTop) (the maximum is raised lazily, by 2^8), which leaves f16 probabilities
    // 2^-30 of the largest before they are lost; bf16 has f32's range.
    constexpr float kTop = F16 ? 6.0f : 0.0f;

    stage(0);
    if (n_tile > 1) fetch(KT);
    __syncthreads();
    for (int w = 0; w < n_tile; w++) {
        const int buf = w & 1, base = w * KT;
        const u32x4 *kb = kt + buf * KT * CPR, *vb = vt + buf * KT * CPR;
        if (w + 1 < n_tile) stage(buf ^ 1);
        if (w + 2 < n_tile) fetch(base + 2 * KT);
        if (base <= qmax_w) {
            floatx16 sc[NKB];
#pragma unroll
            for (int b = 0; b < NKB; b++) sc[b] = (floatx16)0.0f;
#pragma unroll
            for (int t = 0; t < NKS; t++)
#pragma unroll
                for (int b = 0; b < NKB; b++) {
                    const int r = 32 * b + j;
                    const V8 kh = __builtin_bit_cast(V8, kb[r * CPR + kslot<CPR>(r, 2 * t + hf)]);
                    sc[b] = mfma(kh, qh[t], sc[b]);
                    if constexpr (NP == 2) {
                        const V8 kl = __builtin_bit_cast(V8, kb[r * CPR + kslot<CPR>(r, HD / 8 + 2 * t + hf)]);
                        sc[b] = mfma(kh, ql[t], sc[b]);
                        sc[b] = mfma(kl, qh[t], sc[b]);
                    }
                }
            // scores in the exp2 domain: x = s scale (K's row scale folded in)
            const bool mask = base + KT - 1 > qmin_w;
            const float *ke = se + buf * 2 * KT, *ve = ke + KT;
            float mloc = -INFINITY;
            bool odd_rows = false;  // two planes: a value row of the tile is not finite (its K scale is negative)
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    floatx4 k4 = (floatx4)qscale, v4 = (floatx4)0.0f;
                    if constexpr (NP == 2) {
                        const floatx4 s4 = *reinterpret_cast<const floatx4 *>(ke + 32 * b + 8 * q + 4 * hf);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            odd_rows |= s4[r] < 0.0f;
                            k4[r] = qscale * fabsf(s4[r]);
                        }
                        v4 = *reinterpret_cast<const floatx4 *>(ve + 32 * b + 8 * q + 4 * hf);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float x = sc[b][4 * q + r] * k4[r];
                        if constexpr (SOFTCAP) {
                            x = tanhf(x / a.softcap) * (a.softcap * kLog2e);
                        }
                        // (two planes: the weight that P has to carry is p 2^ve)
                        if constexpr (NP == 2) x += v4[r];
                        if (mask && base + 32 * b + 8 * q + 4 * hf + r > qpos) x = -INFINITY;
                        sc[b][4 * q + r] = x;
                        mloc = fmaxf(mloc, x);
                    }
                }
            mloc = both_max(mloc);
            if (__builtin_amdgcn_ballot_w64(mloc - m_run > 8.0f) != 0) {
                const float m_new = mloc - m_run > 8.0f ? mloc : m_run;
                const float alpha = exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < NDB; db++) o[db] *= alpha;
            }
            const float off = kTop - m_run;
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    floatx4 v4 = (floatx4)0.0f;
                    if constexpr (NP == 2) v4 = *reinterpret_cast<const floatx4 *>(ve + 32 * b + 8 * q + 4 * hf);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float p = __builtin_amdgcn_exp2f(sc[b][4 * q + r] + off);
                        sc[b][4 * q + r] = p;
                        l_run += NP == 2 ? p * __builtin_amdgcn_exp2f(-v4[r]) : p;
                    }
                }
#pragma unroll
            for (int st = 0; st < 2 * NKB; st++) {
                V8 pb, pl;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = sc[st >> 1][8 * (st & 1) + e];
                    pb[e] = (T)p;
                    if constexpr (NP == 2) pl[e] = (T)(p - (float)pb[e]);
                }
                V8 va[NDB], vl[NP == 2 ? NDB : 1];
#pragma unroll
                for (int db = 0; db < NDB; db++) {
                    va[db] = v_operand<T, CPR>(vb, 16 * st, 4 * db, lane);
                    if constexpr (NP == 2) vl[db] = v_operand<T, CPR>(vb, 16 * st, HD / 8 + 4 * db, lane);
                }
                if (mask || NP == 2) {
                    // 0 times an infinite or NaN value must not reach the sums (0: a masked key's P, or the low
                    // part of any): what is not finite is added apart, where a visible key brings it.
                    bool bad = odd_rows;
                    if constexpr (NP == 1) {
#pragma unroll
                        for (int db = 0; db < NDB; db++) bad |= any_bad(va[db], F16);
                    }
                    if (__builtin_amdgcn_ballot_w64(bad) != 0) {
                        V8 see;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int key = base + 16 * st + 8 * (e >> 2) + 4 * hf + (e & 3);
                            see[e] = key <= qpos ? (T)1.0f : (T)0.0f;
                        }
#pragma unroll
                        for (int db = 0; db < NDB; db++) {
                            const floatx16 up = mfma(bad_part<T>(va[db], 1), see, (floatx16)0.0f);
                            const floatx16 dn = mfma(bad_part<T>(va[db], 2), see, (floatx16)0.0f);
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                o[db][e] += up[e] > 0.0f ? INFINITY : 0.0f;
                                o[db][e] -= dn[e] > 0.0f ? INFINITY : 0.0f;
                            }
                            va[db] = bad_part<T>(va[db], 0);
                            if constexpr (NP == 2) vl[db] = bad_part<T>(vl[db], 0);
                        }
                    }
                }
#pragma unroll
                for (int db = 0; db < NDB; db++) {
                    o[db] = mfma(va[db], pb, o[db]);
                    if constexpr (NP == 2) {
                        o[db] = mfma(va[db], pl, o[db]);
                        o[db] = mfma(vl[db], pb, o[db]);
                    }
                }
            }
        }
        __syncthreads();
    }

    const float inv = 1.0f / both_sum(l_run);
    O *orow = static_cast<O *>(a.out) + (row0 + tok) * a.os + (int64_t)head * hd;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++) {
            // this lane half's 8 consecutive dims: 32 db + 16 q2 + 8 hf ..
            float x[8];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[db][8 * q2 + r] * inv),
                                                          __float_as_uint(o[db][8 * q2 + 4 + r] * inv), false, false);
                x[r] = __uint_as_float(s[0]);
                x[4 + r] = __uint_as_float(s[1]);
            }
            const int d = 32 * db + 16 * q2 + 8 * hf;
            if (live && d < hd) store8(orow + d, x);
        }
}

// f32 K and V rows into two f16 planes: x 2^-e = hi + lo with the row's largest |x| 2^-e in [2^13, 2^14),
// hi rounded, lo the rest rounded (below 2^2: kept to 2^-9 of it and more).  K's scale is 2^e; of V's
// the exponent e is kept.  A row of zeros, or one that is not finite throughout, has e = 0 (hi then
// holds its infinities and NaN); a row of zeros of V e = -64, so that it claims no range of P.
// A V row with an element that is not finite makes the K scale of its token negative.
// One thread per 8 dims of a row, a row's threads in one wave.
template <int HD>
__global__ __launch_bounds__(256) void prompt_split_kernel(const float *__restrict__ k, int64_t ks,
                                                           const float *__restrict__ v, int64_t vs, int64_t row0,
                                                           int64_t n_rows, int H, int hd, _Float16 *kp, _Float16 *vp,
                                                           float *ke, float *ve) {
    constexpr int LPR = HD / 8;
    const int64_t idx = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
    const int l = threadIdx.x % LPR;
    if (idx >= n_rows * H) return;
    const int64_t row = idx / H;
    const int h = (int)(idx - row * H);
    const bool in = 8 * l < hd;
    float kscale = 1.0f;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const float *src = which ? v + (row0 + row) * vs : k + (row0 + row) * ks;
        float x[8];
        load8(src + (int64_t)h * hd + (in ? 8 * l : 0), x);
        float m = 0.0f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = in ? x[e] : 0.0f;
            m = fmaxf(m, fabsf(x[e]));
            bad |= !(fabsf(x[e]) < INFINITY);
        }
        m = bad ? INFINITY : m;
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        int e2 = 0;
        if (m > 0.0f && m < INFINITY) e2 = max(ilogbf(m), -100) - 13;
        const float s = ldexpf(1.0f, -e2);
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = opaque(x[e] * s);
            hi[e] = (_Float16)y;
            const float rest = y - (float)hi[e];
            lo[e] = fabsf(y) < INFINITY && fabsf((float)hi[e]) < INFINITY ? (_Float16)rest : (_Float16)0.0f;
        }
        _Float16 *dst = (which ? vp : kp) + idx * (2 * HD) + 8 * l;
        *reinterpret_cast<f16x8 *>(dst) = hi;
        *reinterpret_cast<f16x8 *>(dst + HD) = lo;
        if (l == 0) {
            if (which) {
                ve[idx] = m == 0.0f ? -64.0f : (float)e2;
                ke[idx] = m < INFINITY ? kscale : -kscale;
            } else {
                kscale = ldexpf(1.0f, e2);
            }
        }
    }
}

template <class T, class O, int HD, int NP, int KT, bool SC>
void prompt_launch(const PromptArgs &a, unsigned blocks, hipStream_t st) {
    constexpr size_t lds = (size_t)4 * KT * NP * HD * 2 + (NP == 2 ? 4 * KT * sizeof(float) : 0);
    static_assert(lds <= 160 * 1024, "the tiles fit a CU's LDS");
    if (lds > 64 * 1024)
        (void)hipFuncSetAttribute((const void *)prompt_kernel<T, O, HD, NP, KT, SC>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    prompt_kernel<T, O, HD, NP, KT, SC><<<blocks, 64 * kPromptNW, lds, st>>>(a);
}

template <class T, class O, int NP>
void prompt_dims(const PromptArgs &a, bool cap, unsigned blocks, hipStream_t st) {
    if (a.hd <= 64) {
        if (cap) prompt_launch<T, O, 64, NP, 64, true>(a, blocks, st);
        else prompt_launch<T, O, 64, NP, 64, false>(a, blocks, st);
    } else if (a.hd <= 128) {
        if (cap) prompt_launch<T, O, 128, NP, 64 / NP, true>(a, blocks, st);
        else prompt_launch<T, O, 128, NP, 64 / NP, false>(a, blocks, st);
    } else {
        if (cap) prompt_launch<T, O, 256, NP, 32, true>(a, blocks, st);
        else prompt_launch<T, O, 256, NP, 32, false>(a, blocks, st);
    }
}

int padded(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

}  // namespace

uint64_t prompt_workspace(int32_t dtype, int64_t n_rows, int n_kv, int hd) {
    if (dtype != TS_DTYPE_F32) return 0;
    return (uint64_t)n_rows * n_kv * (2 * 2 * 2 * (uint64_t)padded(hd) + 8);
}

hipError_t launch_prompt(const PromptCall &c, hipStream_t st) {
    PromptArgs a = {};
    a.q = c.q;
    a.k = c.k;
    a.v = c.v;
    a.out = c.out;
    a.qs = c.q_stride;
    a.ks = c.k_stride;
    a.vs = c.v_stride;
    a.os = c.out_stride;
    a.G = c.n_head / c.n_kv;
    a.H = c.n_kv;
    a.hd = c.hd;
    const bool cap = c.softcap > 0.0f;
    a.scale = (cap ? 1.0f : kLog2e) / sqrtf((float)c.hd);
    a.softcap = c.softcap;
    a.row0 = c.off[0];
    if (c.dtype == TS_DTYPE_F32) {
        const int64_t n = c.off[c.n_seq] - c.off[0], rows = n * c.n_kv;
        const int hdp = padded(c.hd);
        _Float16 *kp = static_cast<_Float16 *>(c.ws), *vp = kp + rows * 2 * hdp;
        float *ke = reinterpret_cast<float *>(vp + rows * 2 * hdp), *ve = ke + rows;
        a.kp = kp;
        a.vp = vp;
        a.ke = ke;
        a.ve = ve;
        const unsigned blocks = (unsigned)((rows * (hdp / 8) + 255) / 256);
        const float *k = static_cast<const float *>(c.k), *v = static_cast<const float *>(c.v);
        if (hdp == 64)
            prompt_split_kernel<64><<<blocks, 256, 0, st>>>(k, a.ks, v, a.vs, a.row0, n, c.n_kv, c.hd, kp, vp, ke, ve);
        else if (hdp == 128)
            prompt_split_kernel<128><<<blocks, 256, 0, st>>>(k, a.ks, v, a.vs, a.row0, n, c.n_kv, c.hd, kp, vp, ke, ve);
        else
            prompt_split_kernel<256><<<blocks, 256, 0, st>>>(k, a.ks, v, a.vs, a.row0, n, c.n_kv, c.hd, kp, vp, ke, ve);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int G = a.G;
    for (int s = 0; s < c.n_seq; s += a.t.n) {
        pack_fill(a.t, c.off, nullptr, c.n_seq, s,
                  [G](int n) { return (int)(((int64_t)n * G + kPromptCols - 1) / kPromptCols); });
        const int64_t blocks = (int64_t)a.t.item[a.t.n] * c.n_kv;
        if (blocks == 0) continue;
        if (c.dtype == TS_DTYPE_F32)
            prompt_dims<_Float16, float, 2>(a, cap, (unsigned)blocks, st);
        else if (c.dtype == TS_DTYPE_F16)
            prompt_dims<_Float16, _Float16, 1>(a, cap, (unsigned)blocks, st);
        else
            prompt_dims<__bf16, __bf16, 1>(a, cap, (unsigned)blocks, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ts
