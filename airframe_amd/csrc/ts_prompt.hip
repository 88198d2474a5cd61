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
//
// Matrix work bounds it.  A prompt of 8192 tokens, 32 heads over 8 of 128 dims in f16: 550 GFLOP in 550 to 600 us
// by card, 0.92 to 1.00 PFLOP/s (a product of 8192^3 reaches 1.15), the matrix cores busy for 54% of the CUs' time
// and no bank conflicts.  16 ragged prompts of 300 to 2048 in bf16, 150 GFLOP: 202 us; f32 (three products) of 128 dims
// 560 us, of 64 dims 315.  3 prompts of 501 to 2100, 16 heads over 8 of 256 dims in f32 with softcap: 265 us behind 18 of
// the split, one wave per SIMD (o alone takes 128 registers), ended by the longest walk of 66 tiles (26 on
// average): 0.53 PFLOP/s of the three products' work.
#include "ts_prompt.h"

#include <cfloat>
#include <type_traits>

#include "ts_mfma.h"

namespace ts {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));

constexpr int kPromptNW = 4;
constexpr int kPromptCols = 32 * kPromptNW;
constexpr float kFar = 4194304.0f;   // scores above this: their reference is taken from them first
constexpr int kLowest = -113;         // f32: least exponent that rows are scaled by (2^(13 - it) and its inverse are normal)
constexpr float kZeroRow = -200.0f;  // f32: V's exponent of a row of zeros (below any other: out of P's range)

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
    float softcap, inv_softcap;  // (inv_softcap: cap_quick's to_exp where that is taken)
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

// The 8 keys of one lane of a 16-key step, of one dim: 4 rows at p and 4 rows 8 further on.  Each group
// of 16 lanes points at 4 rows x 16 dims and gets them transposed.
template <class T, int ROWB>
__device__ inline typename Vec8<T>::type v_operand(const unsigned char *p) {
    typedef __attribute__((address_space(3))) short4v *lds4;
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 8 * ROWB));
    const short8v s = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(typename Vec8<T>::type, s);
}

// softcap tanh(x / softcap) in the exp2 domain, within 2^-20 of it relative to it for any softcap: with y = x /
// softcap, x (1 + y^2 P(y^2)) near zero, P fitted to (tanh(y) / y - 1) / y^2 by least squares on Chebyshev nodes, and
// softcap (1 - 2 / (1 + e^(2 y))) beyond, whose error is 2^-22 of softcap and not of x; the two are
// selected, not branched to.  f32 rows: P of five terms below 0.6 (2^-27), 16-bit rows, whose weights are rounded to
// 2^-12 and 2^-9, of three below 0.35 (2^-24).
template <bool F32>
__device__ inline float cap(float x, float softcap, float inv_softcap) {
    const float y = x * inv_softcap, z = y * y, xl = x * kLog2e;
    float p;
    if constexpr (F32) {
        p = __builtin_fmaf(z, -5.8939453e-03f, 2.0794618e-02f);
        p = __builtin_fmaf(z, p, -5.3783293e-02f);
        p = __builtin_fmaf(z, p, 1.3331915e-01f);
        p = __builtin_fmaf(z, p, -3.33332975e-01f);
    } else {
        p = __builtin_fmaf(z, -4.9134325e-02f, 1.3299560e-01f);
        p = __builtin_fmaf(z, p, -3.33326515e-01f);
    }
    const float near = __builtin_fmaf(xl * z, p, xl);
    const float rest = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * (2.0f * kLog2e)) + 1.0f);
    const float far = softcap * __builtin_fmaf(-2.0f * kLog2e, rest, kLog2e);
    return fabsf(y) < (F32 ? 0.6f : 0.35f) ? near : far;
}

// The same of small softcaps for 16-bit rows, as c - 2 c / (1 + e^(2 y)) from two transcendental instructions: within
// 2^-21 of softcap and not of x, so up to softcaps of kQuickCap within 2^-15, where f16 weights are rounded by 2^-12.
// to_exp: 2 log2(e) / softcap.  16 ragged prompts, softcap 50, with this and with cap(): bf16 of 128 dims 236 and 293 us,
// f16 of 64 dims 153 and 226 (without softcap 202 and 109).
constexpr float kQuickCap = 64.0f;
__device__ inline float cap_quick(float x, float softcap, float to_exp) {
    const float c = softcap * kLog2e;
    return c - 2.0f * c * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * to_exp) + 1.0f);
}

// The largest exponent bits of packed 16-bit floats: m and those of v, and whether they are an infinity's or
// a NaN's.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <class V>
__device__ inline void max_bits(u16x2 &m, V v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
}
__device__ inline bool not_finite(u16x2 m, bool f16) { return max(m[0], m[1]) >= (f16 ? 0x7C00 : 0x7F80); }
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

// One tile of 64 lanes x 16 bytes from memory straight into LDS: lane l's 16 bytes at byte voff of the
// buffer (0s past its end) go to lds + 16 l.  In asm because the compiler would make every LDS read
// wait for all such loads; it has no outputs but M0's old value (put back: the compiler may hold one of its own
// there), and tile_barrier() waits for it.
__device__ inline void load_lds(const u32x4 &rsrc, uint32_t voff, uint32_t lds) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(voff), "s"(rsrc), "s"(lds) : "memory");
}
// All loads into LDS of this wave have landed, and every wave of the workgroup got here.
__device__ inline void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A buffer of `bytes` from p on (2^31 at most: no offset into it is larger); reads past it give 0.
__device__ inline u32x4 buffer_of(const void *p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    u32x4 r = {(uint32_t)a, (uint32_t)(a >> 32) & 0xFFFFu, (uint32_t)min(bytes, (int64_t)0x80000000), 0x00027000u};
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
}

// T: the matrix cores' type; O: the rows' type (float with two planes); HD: head dims, padded; NP:
// planes; KT: keys per tile; CAP: no softcap, cap_quick or cap.
enum { kNoCap = 0, kCapQuick = 1, kCap = 2 };
template <class T, class O, int HD, int NP, int KT, int CAP>
__global__ __launch_bounds__(64 * kPromptNW, HD > 128 ? 1 : 2) void prompt_kernel(PromptArgs a) {
    using V8 = typename Vec8<T>::type;
    constexpr int CPR = NP * HD / 8;  // 16-byte chunks of a tile's row
    constexpr int ROWB = 16 * CPR, TILEB = KT * ROWB;
    constexpr int NKS = HD / 16, NDB = HD / 32, NKB = KT / 32;
    constexpr int NW = kPromptNW, NLD = TILEB / 1024 / NW;  // loads of 1 KB of a tile per wave
    constexpr bool F16 = __is_same(T, _Float16);
    constexpr bool RAW = NP == 1 && CAP == kNoCap;  // scores stay unscaled until the exponent's FMA
    static_assert(TILEB % (1024 * NW) == 0, "a tile's loads spread evenly");
    // [2 buffers] K tile, V tile; then, of two planes, [2][2][KT] K scales and V exponents
    extern __shared__ __align__(1024) unsigned char pr_smem[];
    float *const se = reinterpret_cast<float *>(pr_smem + 4 * TILEB);

    const int item = blockIdx.x / a.H, h = blockIdx.x - item * a.H;
    const int i = pack_find(a.t, item);
    const int row0 = a.t.tok[i], n = a.t.pos0[i];  // (rows of the i-th sequence: pos0)
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

    // Loads of a tile: wave w's p-th takes 1 KB of it, 1024 / ROWB rows; the lane's slot in its row holds
    // the chunk that kslot / vslot put there.
    const uint8_t *kbase, *vbase;
    int64_t kstride, vstride;  // bytes from key to key
    if constexpr (NP == 1) {
        kbase = reinterpret_cast<const uint8_t *>(static_cast<const T *>(a.k) + (int64_t)row0 * a.ks + (int64_t)h * hd);
        vbase = reinterpret_cast<const uint8_t *>(static_cast<const T *>(a.v) + (int64_t)row0 * a.vs + (int64_t)h * hd);
        kstride = 2 * a.ks;
        vstride = 2 * a.vs;
    } else {
        const int64_t at = ((row0 - a.row0) * a.H + h) * (int64_t)(NP * HD);
        kbase = reinterpret_cast<const uint8_t *>(a.kp + at);
        vbase = reinterpret_cast<const uint8_t *>(a.vp + at);
        kstride = vstride = (int64_t)a.H * ROWB;
    }
    uint32_t ko[NLD], vo[NLD];
#pragma unroll
    for (int p = 0; p < NLD; p++) {
        const int at = 64 * (wave + NW * p) + lane, r = at / CPR, s = at % CPR;
        const int kc = kslot<CPR>(r, s), vc = vslot<CPR>(r, s);  // (an XOR: its own inverse)
        // chunks past the row are read past the buffer's end: zeros
        ko[p] = NP == 2 || kc < n_chunk ? (uint32_t)(r * kstride) + 16 * kc : 0xFFFFFFF0u;
        vo[p] = NP == 2 || vc < n_chunk ? (uint32_t)(r * vstride) + 16 * vc : 0xFFFFFFF0u;
    }
    const int row_bytes = NP == 2 ? ROWB : 2 * hd;
    float pe = 0.0f;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)pr_smem;
    auto fetch = [&](int w, int buf) __attribute__((always_inline)) {
        // (keys past the sequence's end read as zeros; they are masked)
        const int left = n - w * KT;
        const u32x4 kr = buffer_of(kbase + w * KT * kstride, (left - 1) * kstride + row_bytes);
        const u32x4 vr = buffer_of(vbase + w * KT * vstride, (left - 1) * vstride + row_bytes);
        const uint32_t to = lds0 + buf * 2 * TILEB + 1024 * wave;
#pragma unroll
        for (int p = 0; p < NLD; p++) load_lds(kr, ko[p], to + 1024 * NW * p);
#pragma unroll
        for (int p = 0; p < NLD; p++) load_lds(vr, vo[p], to + TILEB + 1024 * NW * p);
        if constexpr (NP == 2)
            if (tid < 2 * KT) {
                const int64_t at = (row0 - a.row0 + min(w * KT + tid % KT, n - 1)) * a.H + h;
                pe = tid < KT ? a.ke[at] : a.ve[at];
            }
    };
    fetch(0, 0);
    if constexpr (NP == 2)
        if (tid < 2 * KT) se[tid] = pe;

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
        // the largest element to [2^13, 2^14), as the planes' rows (and below, from 2^-113 on)
        m = both_max(m);
        const int e2 = m > 0.0f ? min(max(ilogbf(m), kLowest), 127) - 13 : 0;
        const float s = ldexpf(1.0f, -e2);
        qscale = a.scale * ldexpf(1.0f, e2);
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

    // This lane's operand addresses in a tile: K chunk 2 t + hf of row j (rows 32 and more further on),
    // V rows 4 hf + i / 4 (transposed in groups of 16 lanes), dims of tile db.
    // The XORs reach 16 chunks: what lies further on is 256 bytes and more away from one of the first.
    constexpr int NKA = NKS < 8 ? NKS : 8, NVA = NDB < 4 ? NDB : 4;
    uint32_t ka[NKA], va_[NVA];
#pragma unroll
    for (int t = 0; t < NKA; t++) ka[t] = j * ROWB + 16 * kslot<CPR>(j, 2 * t + hf);
#pragma unroll
    for (int db = 0; db < NVA; db++) {
        const int l = lane & 15, r = 4 * hf + (l >> 2), ch = 4 * db + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1);
        va_[db] = r * ROWB + 16 * vslot<CPR>(r, ch) + 8 * (l & 1);
    }
    // (64 dims in two planes are one row of 16 chunks: t and db of the low plane start in its middle)
    auto k_at = [&](int t) { return HD == 64 && t >= NKS ? ka[t - NKS] ^ 128 : ka[t & (NKA - 1)] + t / NKA * 256; };
    auto v_at = [&](int db) { return HD == 64 && db >= NDB ? va_[db - NDB] ^ 128 : va_[db & (NVA - 1)] + db / NVA * 256; };

    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) o[db] = (floatx16)0.0f;
    // The softmax's reference: below every finite score, the first tile sets it.  Of two planes that of the scores,
    // and l_run's; P, which carries the value rows' sizes too, has o_rel above it.
    float m_run = -3.4e38f, l_run = 0.0f;
    float o_rel = -3.4e38f;
    // P is held up to 2^(8 + kTop) (the maximum is raised lazily, by 2^8), which leaves f16 probabilities
    // 2^-30 of the largest before they are lost; bf16 has f32's range.
    constexpr float kTop = F16 ? 6.0f : 0.0f;

    auto tile = [&](auto MASKED, int w) __attribute__((always_inline)) {
        constexpr bool MASK = decltype(MASKED)::value;
        const int base = w * KT;
        const unsigned char *kb = pr_smem + (w & 1) * 2 * TILEB, *vb = kb + TILEB;
        floatx16 sc[NKB];
#pragma unroll
        for (int b = 0; b < NKB; b++) sc[b] = (floatx16)0.0f;
        // (the next k-step's operands are read beside this one's products, and no further ahead: left to
        // itself the compiler reads the whole tile first and spills)
        V8 kf[2][NKB][NP];
        auto read_k = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int pl = 0; pl < NP; pl++)
                    kf[t & 1][b][pl] = *reinterpret_cast<const V8 *>(kb + k_at(pl * NKS + t) + 32 * b * ROWB);
        };
        read_k(0);
#pragma unroll
        for (int t = 0; t < NKS; t++) {
            if (t + 1 < NKS) read_k(t + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 0; b < NKB; b++) sc[b] = mfma(kf[t & 1][b][0], qh[t], sc[b]);
            if constexpr (NP == 2) {
#pragma unroll
                for (int b = 0; b < NKB; b++) sc[b] = mfma(kf[t & 1][b][0], ql[t], sc[b]);
#pragma unroll
                for (int b = 0; b < NKB; b++) sc[b] = mfma(kf[t & 1][b][NP - 1], qh[t], sc[b]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // x: scores in the exp2 domain; without softcap and planes their scale waits for the exponent's FMA.
        const float *ke = se + (w & 1) * 2 * KT, *ve = ke + KT;
        // Two planes: K or V of a key in the tile are not finite (its K scale is negative).  The planes hold 0 for those
        // elements: hi and lo terms of an infinity would meet as NaN.  What they bring is added apart, to the
        // scores here and to the sums below.
        bool odd_rows = false;
        if constexpr (NP == 2) odd_rows = __builtin_amdgcn_ballot_w64(ke[lane % KT] < 0.0f) != 0;
        if (odd_rows) {
            const float *qr = static_cast<const float *>(a.q) + (row0 + tok) * a.qs + (int64_t)head * hd;
#pragma unroll 1
            for (int kk = 0; kk < KT; kk++) {
                if (base + kk >= n || __builtin_amdgcn_readfirstlane(__float_as_int(ke[kk])) >= 0) continue;
                const float *kr = static_cast<const float *>(a.k) + (int64_t)(row0 + base + kk) * a.ks + (int64_t)h * hd;
                float extra = 0.0f;
#pragma unroll 1
                for (int d = 8 * hf; d < hd; d += 16)
#pragma unroll
                    for (int e = 0; e < 8; e++) extra += !(fabsf(kr[d + e]) < INFINITY) ? qr[d + e] * kr[d + e] : 0.0f;
                extra = both_sum(extra);
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] += 32 * b + 8 * (e >> 2) + 4 * hf + (e & 3) == kk ? extra : 0.0f;
            }
        }
        float mloc = -INFINITY;
#pragma unroll
        for (int b = 0; b < NKB; b++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                floatx4 k4 = (floatx4)qscale;
                if constexpr (NP == 2) {
                    const floatx4 s4 = *reinterpret_cast<const floatx4 *>(ke + 32 * b + 8 * q + 4 * hf);
#pragma unroll
                    for (int r = 0; r < 4; r++) k4[r] = qscale * fabsf(s4[r]);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = sc[b][4 * q + r];
                    if constexpr (!RAW) x = opaque(x * k4[r]);  // (rounded in every tile: an FMA with the reference in some is not)
                    if constexpr (CAP == kCapQuick) x = cap_quick(x, a.softcap, a.inv_softcap);
                    if constexpr (CAP == kCap) x = cap<NP == 2>(x, a.softcap, a.inv_softcap);
                    if constexpr (MASK)
                        if (base + 32 * b + 8 * q + 4 * hf + r > qpos) x = -INFINITY;
                    sc[b][4 * q + r] = x;
                    mloc = fmaxf(mloc, x);
                }
            }
        mloc = both_max(mloc);
        if constexpr (RAW) mloc *= qscale;
        if constexpr (NP == 2) mloc = ceilf(mloc);
        if (__builtin_amdgcn_ballot_w64(mloc - m_run > 8.0f) != 0) {
            const float m_new = mloc - m_run > 8.0f ? mloc : m_run, d = m_run - m_new;
            const float alpha = exp2f(d);
            m_run = m_new;
            l_run *= alpha;
            if constexpr (NP == 2) {
                o_rel += d;
            } else {
#pragma unroll
                for (int db = 0; db < NDB; db++) o[db] *= alpha;
            }
        }
        // Two planes: P carries 2^(x + ve - o's reference), the probability times its value row's size, and has a maximum
        // of its own.  The reference of the scores is taken from them first, so that what ve is added to is small where it
        // counts, whatever their size; all references are whole numbers, as ve is, and moving them is exact.
        if constexpr (NP == 2) {
            float ploc = -INFINITY;
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const floatx4 v4 = *reinterpret_cast<const floatx4 *>(ve + 32 * b + 8 * q + 4 * hf);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        sc[b][4 * q + r] -= m_run;
                        ploc = fmaxf(ploc, sc[b][4 * q + r] + v4[r]);
                    }
                }
            ploc = ceilf(both_max(ploc));
            if (__builtin_amdgcn_ballot_w64(ploc - o_rel > 8.0f) != 0) {
                const float o_new = ploc - o_rel > 8.0f ? ploc : o_rel;
                const float alpha = exp2f(o_rel - o_new);
                o_rel = o_new;
#pragma unroll
                for (int db = 0; db < NDB; db++) o[db] *= alpha;
            }
        }
        if constexpr (NP == 2)
            if (odd_rows) {
                // value rows that are not finite: a key that a column sees brings those elements as they are
#pragma unroll 1
                for (int kk = 0; kk < KT; kk++) {
                    if (base + kk >= n || __builtin_amdgcn_readfirstlane(__float_as_int(ke[kk])) >= 0) continue;
                    const float *vr = static_cast<const float *>(a.v) + (int64_t)(row0 + base + kk) * a.vs + (int64_t)h * hd;
#pragma unroll
                    for (int db = 0; db < NDB; db++)
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int d = 32 * db + 8 * q + 4 * hf;
                            const floatx4 x = *reinterpret_cast<const floatx4 *>(vr + (d < hd ? d : 0));
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                o[db][4 * q + r] += base + kk <= qpos && !(fabsf(x[r]) < INFINITY) ? x[r] : 0.0f;
                        }
                }
            }
        // One plane: a weight is 2^(pmul x + off).  Below 2^22 that is one FMA of the scores as they are.  Above, the FMA's
        // exact product and the rounded reference would be up to half a step of the reference apart (1024 at 2^34),
        // and off would lose kTop: the scores are rounded, and the reference taken from them first.
        float pmul = qscale, off = kTop - (NP == 2 ? o_rel : m_run);
        if constexpr (NP == 1)
            if (__builtin_amdgcn_ballot_w64(m_run > kFar || (m_run < -kFar && m_run > -3.0e38f)) != 0) {
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[b][e] = opaque(RAW ? sc[b][e] * qscale : sc[b][e]) - m_run;
                pmul = 1.0f;
                off = kTop;
            }
        // O^T += V^T P^T, 16 keys at a time: the exponentials of a step run beside the products of the one
        // before, and V's operands are read one group of products ahead.  (Two planes: one dim tile a group, or
        // 128 dims take more than the 256 registers that let two workgroups share a CU: 1006 against 560 us for
        // 16 f32 prompts of 300-2048 tokens; 64 dims 349 and 315.)
        constexpr int VG = NP == 2 ? 1 : 4, NVG = NDB < VG ? 1 : NDB / VG, NU = 2 * NKB * NVG;
        constexpr int DG = NDB < VG ? NDB : VG;  // dim tiles of a group
        V8 vf[2][DG][NP];
        auto read_v = [&](int u) __attribute__((always_inline)) {
#pragma unroll
            for (int d = 0; d < DG; d++)
#pragma unroll
                for (int pl = 0; pl < NP; pl++)
                    vf[u & 1][d][pl] = v_operand<T, ROWB>(vb + v_at(pl * NDB + DG * (u % NVG) + d) + 16 * (u / NVG) * ROWB);
        };
        read_v(0);
        V8 pb, pl;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const int st = u / NVG;
            if (u % NVG == 0) {
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    floatx4 v4 = (floatx4)0.0f;
                    if constexpr (NP == 2) v4 = *reinterpret_cast<const floatx4 *>(ve + 16 * st + 8 * q + 4 * hf);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float x = sc[st >> 1][8 * (st & 1) + 4 * q + r];
                        const float p = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(x, pmul, off) : x + (v4[r] + off));
                        l_run += NP == 2 ? __builtin_amdgcn_exp2f(x) : p;
                        const T hi = (T)p;
                        pb[4 * q + r] = hi;
                        if constexpr (NP == 2) pl[4 * q + r] = (T)(p - (float)hi);
                    }
                }
            }
            V8 (&va)[DG][NP] = vf[u & 1];
            floatx16 *const og = o + DG * (u % NVG);
            if (u + 1 < NU) read_v(u + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (MASK && NP == 1) {
                // 0 times an infinite or NaN value of a masked key must not reach the sums: what is not finite is
                // added apart, where a visible key brings it.
                u16x2 bits = {0, 0};
#pragma unroll
                for (int d = 0; d < DG; d++) max_bits(bits, va[d][0]);
                const bool bad = not_finite(bits, F16);
                if (__builtin_amdgcn_ballot_w64(bad) != 0) {
                    V8 see;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int key = base + 16 * st + 8 * (e >> 2) + 4 * hf + (e & 3);
                        see[e] = key <= qpos ? (T)1.0f : (T)0.0f;
                    }
#pragma unroll
                    for (int d = 0; d < DG; d++) {
#pragma unroll
                        for (int sign = 1; sign <= 2; sign++) {
                            const floatx16 hit = mfma(bad_part<T>(va[d][0], sign), see, (floatx16)0.0f);
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                og[d][e] += hit[e] > 0.0f ? (sign == 1 ? INFINITY : -INFINITY) : 0.0f;
                        }
                        // (in place: these operands are not used again)
                        va[d][0] = bad_part<T>(va[d][0], 0);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < DG; d++) og[d] = mfma(va[d][0], pb, og[d]);
            if constexpr (NP == 2) {
#pragma unroll
                for (int d = 0; d < DG; d++) og[d] = mfma(va[d][0], pl, og[d]);
#pragma unroll
                for (int d = 0; d < DG; d++) og[d] = mfma(va[d][NP - 1], pb, og[d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Tiles that every column of the wave sees whole, then those on its diagonal.  (Two loops: with both
    // bodies in one, the compiler moves the accumulators between them.)  Every wave passes n_tile barriers.
    auto step = [&](auto MASKED, int w, bool busy) __attribute__((always_inline)) {
        tile_barrier();  // tile w is there; nobody reads tile w - 1 any more
        if (w + 1 < n_tile) fetch(w + 1, (w + 1) & 1);
        if (busy) tile(MASKED, w);
        if constexpr (NP == 2)
            if (w + 1 < n_tile && tid < 2 * KT) se[((w + 1) & 1) * 2 * KT + tid] = pe;
    };
    const int n_full = qmax_w < 0 ? 0 : min((qmin_w + 1) / KT, n_tile);
    int w = 0;
    for (; w < n_full; w++) step(std::false_type(), w, true);
    for (; w < n_tile; w++) step(std::true_type(), w, w * KT <= qmax_w);

    const float inv = 1.0f / both_sum(l_run);
    // this lane half's 8 consecutive dims 32 db + 16 q2 + 8 hf .. of its column
    auto dims8 = [&](int db, int q2, float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[db][8 * q2 + r] * inv),
                                                      __float_as_uint(o[db][8 * q2 + 4 + r] * inv), false, false);
            x[r] = __uint_as_float(s[0]);
            x[4 + r] = __uint_as_float(s[1]);
        }
        if constexpr (NP == 2) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = ldexpf(x[e], (int)o_rel - 13 - (int)kTop);
        }
    };
    O *orow = static_cast<O *>(a.out) + (row0 + tok) * a.os + (int64_t)head * hd;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++) {
            float x[8];
            dims8(db, q2, x);
            const int d = 32 * db + 16 * q2 + 8 * hf;
            if (live && d < hd) store8(orow + d, x);
        }
}

// f32 K and V rows into two f16 planes: x 2^-e = hi + lo with the row's largest |x| 2^-e in [2^13, 2^14),
// hi rounded, lo the rest rounded (below 2^2: kept to 2^-9 of it and more).  K's scale is 2^e; of V's
// the exponent e + 13, about log2 of its largest element, is kept (kZeroRow for a row of zeros).  Elements that are not
// finite become 0, and the K scale of their token is made negative.
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
    int bad = 0;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const float *src = which ? v + (row0 + row) * vs : k + (row0 + row) * ks;
        float x[8];
        load8(src + (int64_t)h * hd + (in ? 8 * l : 0), x);
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = in ? x[e] : 0.0f;
            const bool fin = fabsf(x[e]) < INFINITY;
            bad |= !fin;
            x[e] = fin ? x[e] : 0.0f;
            m = fmaxf(m, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) {
            m = fmaxf(m, __shfl_xor(m, o, 64));
            bad |= __shfl_xor(bad, o, 64);
        }
        int e2 = 0;
        if (m > 0.0f) e2 = max(ilogbf(m), kLowest) - 13;
        const float s = ldexpf(1.0f, -e2);
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = opaque(x[e] * s);
            hi[e] = (_Float16)y;
            lo[e] = (_Float16)(y - (float)hi[e]);
        }
        _Float16 *dst = (which ? vp : kp) + idx * (2 * HD) + 8 * l;
        *reinterpret_cast<f16x8 *>(dst) = hi;
        *reinterpret_cast<f16x8 *>(dst + HD) = lo;
        if (l == 0) {
            if (which) {
                ve[idx] = m == 0.0f ? kZeroRow : (float)(e2 + 13);
                ke[idx] = bad ? -kscale : kscale;
            } else {
                kscale = ldexpf(1.0f, e2);
            }
        }
    }
}

template <class T, class O, int HD, int NP, int KT, int CAP>
void prompt_launch(const PromptArgs &a, unsigned blocks, hipStream_t st) {
    constexpr size_t lds = (size_t)4 * KT * NP * HD * 2 + (NP == 2 ? 4 * KT * sizeof(float) : 0);
    static_assert(lds <= 160 * 1024, "the tiles fit a CU's LDS");
    if (lds > 64 * 1024)
        (void)hipFuncSetAttribute((const void *)prompt_kernel<T, O, HD, NP, KT, CAP>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    prompt_kernel<T, O, HD, NP, KT, CAP><<<blocks, 64 * kPromptNW, lds, st>>>(a);
}

// Keys per tile: 64 of one plane and 32 of two up to 128 dims, 32 of 256 dims.  16 ragged prompts of 300 to
// 2048, 32 heads over 8: bf16 of 128 dims 202 us with 64 and 228 with 32, f16 of 64 dims 109 and 130; f32 of 64
// dims 332 with 64 and 315 with 32 (one prompt of 500: 30 and 34; of 8192: 970 and 959), of 128 dims 1382 and
// 560; bf16 of 256 dims 465 with 64 and 467 with 32 (half the LDS).
template <class T, class O, int NP, int CAP>
void prompt_dims(const PromptArgs &a, unsigned blocks, hipStream_t st) {
    if (a.hd <= 64)
        prompt_launch<T, O, 64, NP, 64 / NP, CAP>(a, blocks, st);
    else if (a.hd <= 128)
        prompt_launch<T, O, 128, NP, 64 / NP, CAP>(a, blocks, st);
    else
        prompt_launch<T, O, 256, NP, 32, CAP>(a, blocks, st);
}
template <class T, class O, int NP>
void prompt_cap(const PromptArgs &a, int cap, unsigned blocks, hipStream_t st) {
    if (cap == kNoCap)
        prompt_dims<T, O, NP, kNoCap>(a, blocks, st);
    else if (NP == 2 || cap == kCap)
        prompt_dims<T, O, NP, kCap>(a, blocks, st);
    else if constexpr (NP == 1)
        prompt_dims<T, O, NP, kCapQuick>(a, blocks, st);
}

// Sequences seq0 .. of the batch with the longest first, so that the launch ends with short walks (tok:
// the first row, pos0: the rows).
void fill_longest_first(PackTable &t, const int32_t *off, int n_seq, int seq0, int G) {
    int order[kPackSeqs];
    t.seq0 = seq0;
    t.n = std::min(n_seq - seq0, kPackSeqs);
    for (int i = 0; i < t.n; i++) order[i] = seq0 + i;
    auto len = [&](int s) { return off[s + 1] - off[s]; };
    std::sort(order, order + t.n, [&](int x, int y) { return len(x) != len(y) ? len(x) > len(y) : x < y; });
    t.item[0] = 0;
    for (int i = 0; i < t.n; i++) {
        t.tok[i] = off[order[i]];
        t.pos0[i] = len(order[i]);
        t.item[i + 1] = t.item[i] + (int)(((int64_t)t.pos0[i] * G + kPromptCols - 1) / kPromptCols);
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
    const int cap = c.softcap == 0.0f ? kNoCap : c.dtype != TS_DTYPE_F32 && c.softcap <= kQuickCap ? kCapQuick : kCap;
    a.scale = (cap != kNoCap ? 1.0f : kLog2e) / sqrtf((float)c.hd);
    a.softcap = c.softcap;
    // (finite, so that 0 times it stays 0)
    a.inv_softcap = cap != kNoCap ? std::min((cap == kCapQuick ? 2.0f * kLog2e : 1.0f) / c.softcap, FLT_MAX) : 0.0f;
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
    for (int s = 0; s < c.n_seq; s += a.t.n) {
        fill_longest_first(a.t, c.off, c.n_seq, s, a.G);
        const int64_t blocks = (int64_t)a.t.item[a.t.n] * c.n_kv;
        if (blocks == 0) continue;
        if (c.dtype == TS_DTYPE_F32)
            prompt_cap<_Float16, float, 2>(a, cap, (unsigned)blocks, st);
        else if (c.dtype == TS_DTYPE_F16)
            prompt_cap<_Float16, _Float16, 1>(a, cap, (unsigned)blocks, st);
        else
            prompt_cap<__bf16, __bf16, 1>(a, cap, (unsigned)blocks, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ts
