// ts_weigh.hip -- what every cached slot receives of the attention of new tokens, for gfx950.
//
// For the new tokens t and query heads h of one kv head, P[t,h,p] = softmax over the slots p the token
// sees: w[p] = (w[p]) + sum over t and h of P[t,h,p].  The sums over columns need each softmax's final
// reference and sum, so they come behind the attention itself (one token: ts_weigh_token.hip).
#include "ts_evict.h"
#include "ts_shared.h"
#include "ts_window.h"

namespace ts {

// The attention itself is the window walk of ts_shared.hip over the own keys (its outputs, and every
// column's reference and sum).  Then the columns' rotated q goes into the operand layout of the matrix
// cores once (weigh_prep_kernel), and the scores are computed a second time with the keys held in registers
// and the columns streaming past (weigh_cols_kernel), so that a slot's sum stays in its lane.
namespace {

constexpr int kColBlk = 32;  // columns of one operand block

// One block: q's high halves [k-step][lane][16 bytes], its low terms [group][term][3][lane][8 bytes], then
// q's scale back and the softmax's log2 sum of each column.
template <int HD>
struct ColBlock {
    half8 hi[HD / 16][64];
    uint64_t lo[HD / 64][2][3][64];
    float back[kColBlk], lse[kColBlk];
};

struct ChunkArgs {
    KvLayerView L;
    const int32_t *len;
    const float *q, *rope;
    int rope_pairs, rope_rows, n_head, G, n_tok, n_blk32;
    float inv_sqrt_hd, softcap;
    const float *pm, *pl;  // references and sums of the walk, [rows][slots]
    int slots;
    void *cols;  // [S][H][n_blk32] ColBlock
    int max_seq;
    float *w;
    bool fresh;
};

// 128 columns (token, head) of one kv head and sequence.
template <int HD, bool NORM, bool PAD>
__global__ __launch_bounds__(256) void weigh_prep_kernel(ChunkArgs a) {
    constexpr int NKS = HD / 16, NG = NKS / 4, V4 = HD / 4, QST = HD + 4, BC = 128, NQ = BC * V4 / 256;
    extern __shared__ __align__(16) unsigned char prep_smem[];
    float *const qs = reinterpret_cast<float *>(prep_smem);
    const int h = blockIdx.y, s = blockIdx.z, G = a.G, hdr = PAD ? a.L.hdr : HD, n_cols = a.n_tok * G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j = lane & 31, hf = lane >> 5;
    const int c_blk = blockIdx.x * BC, len = a.len[s];
    const float *const QN = NORM ? a.L.qn : nullptr;
    const float qmul = a.softcap > 0.0f ? a.inv_sqrt_hd : a.inv_sqrt_hd * kLog2e;
#pragma unroll 4
    for (int i = 0; i < NQ; i++) {
        const int at = tid + 256 * i, cl = at / V4, d = 4 * (at % V4);
        const int cg = c_blk + cl, ce = min(cg, n_cols - 1), tok = ce / G;
        const float *qrow = a.q + (((size_t)s * a.n_tok + tok) * a.n_head + h * G + ce % G) * hdr;
        float4 v = keep4(cg < n_cols && d < hdr, *reinterpret_cast<const float4 *>(qrow + (d < hdr ? d : 0)));
        if (QN) {
            float ss = v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
#pragma unroll
            for (int o = 1; o < V4; o <<= 1) ss += __shfl_xor(ss, o, 64);
            const float ns = qk_norm_scale_from_sum(ss, hdr, a.L.norm_eps);
            const float4 w = *reinterpret_cast<const float4 *>(QN + (d < hdr ? d : 0));
            v = make_float4(qk_norm_apply(v.x, ns, w.x), qk_norm_apply(v.y, ns, w.y), qk_norm_apply(v.z, ns, w.z),
                            qk_norm_apply(v.w, ns, w.w));
        }
        const float *rot = a.rope + (size_t)min(rot_of(a.L, s, len + tok), a.rope_rows - 1) * a.rope_pairs * 2;
        if (d / 2 < a.rope_pairs) rope_rotate(v.x, v.y, *reinterpret_cast<const float2 *>(rot + d));
        if (d / 2 + 1 < a.rope_pairs) rope_rotate(v.z, v.w, *reinterpret_cast<const float2 *>(rot + d + 2));
        *reinterpret_cast<float4 *>(qs + cl * QST + d) = v;
    }
    __syncthreads();
    const int b32 = blockIdx.x * 4 + wave;
    if (b32 >= a.n_blk32) return;
    ColBlock<HD> &out = static_cast<ColBlock<HD> *>(a.cols)[((size_t)s * a.L.H + h) * a.n_blk32 + b32];
    const float *const qrow = qs + (32 * wave + j) * QST;
    float mc = 0.0f;
#pragma unroll
    for (int t = 0; t < NKS; t++) {
#pragma unroll
        for (int e = 0; e < 8; e++) mc = fmaxf(mc, fabsf(qrow[8 * (2 * t + hf) + e]));
    }
    float q_s, q_back;
    q_scale(half_max(mc) * qmul, q_s, q_back);
#pragma unroll
    for (int g = 0; g < NG; g++) {
        float lo[32];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int t = 4 * g + u;
            const float *src = qrow + 8 * (2 * t + hf);
            half8 hi;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = opaque(src[kPerm[e]] * (qmul * q_s));
                const _Float16 x = (_Float16)v;
                hi[e] = x;
                lo[8 * u + e] = v - (float)x;
            }
            out.hi[t][lane] = hi;
        }
        int6v t1, t2;
        q_lo_terms(lo, t1, t2);
#pragma unroll
        for (int e = 0; e < 3; e++) {
            out.lo[g][0][e][lane] = (uint32_t)t1[2 * e] | (uint64_t)(uint32_t)t1[2 * e + 1] << 32;
            out.lo[g][1][e][lane] = (uint32_t)t2[2 * e] | (uint64_t)(uint32_t)t2[2 * e + 1] << 32;
        }
    }
    // the softmax's log2 sum over all pieces of the walk
    const int c = c_blk + 32 * wave + j, ce = min(c, n_cols - 1);
    const size_t row = ((size_t)s * a.n_tok + ce / G) * a.n_head + h * G + ce % G;
    float M = kMinit, l = 0.0f;
    for (int i = 0; i < a.slots; i++) M = fmaxf(M, a.pm[row * a.slots + i]);
    for (int i = 0; i < a.slots; i++) {
        const float li = a.pl[row * a.slots + i];
        l += li == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(a.pm[row * a.slots + i] - M) * li;
    }
    if (hf == 0) {
        out.back[j] = q_back;
        out.lse[j] = M + __log2f(l);
    }
}

// Slots of one (sequence, kv head) in blocks of KEYS: wave w of each group of four holds KEYS / 4 keys as
// matrix operands in registers; the two groups take every second column block.  Grid: kv head first, so that the
// workgroups that read one head's columns share an XCD where the heads divide the XCDs.
template <int HD>
constexpr int kColKeys = HD > 128 ? 128 : 256;

template <int HD, bool SOFTCAP>
__global__ __launch_bounds__(512, 2) void weigh_cols_kernel(ChunkArgs a) {
    constexpr int KEYS = kColKeys<HD>, NT = KEYS / 128, NKS = HD / 16, NG = NKS / 4;  // NT: tiles of 32 keys per wave
    extern __shared__ __align__(16) unsigned char cols_smem[];
    using Block = ColBlock<HD>;
    Block *const buf = reinterpret_cast<Block *>(cols_smem);  // [group][2]
    __shared__ float part[2][KEYS];
    const int H = a.L.H, h = blockIdx.x % H, kb = blockIdx.x / H, s = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = wave >> 2, wk = wave & 3;
    const size_t st = (size_t)s * H + h;
    const int len = a.len[s], n = len + a.n_tok, key0 = kb * KEYS;
    float *const w = a.w + st * a.max_seq;
    if (n > a.max_seq) return;  // (a graph replayed past the capacity)
    if (key0 >= n) {
        if (a.fresh)
            for (int p = key0 + tid; p < min(key0 + KEYS, a.max_seq); p += 512) w[p] = 0.0f;
        return;
    }
    const int base = key0 + wk * (KEYS / 4), n_cols = a.n_tok * a.G;
    // (the first columns that see a key of the block; all blocks behind them do too)
    const int first = max(0, key0 - len) * a.G / kColBlk;
    const int n_it = (a.n_blk32 - first + 1) / 2;
    const Block *const src = static_cast<const Block *>(a.cols) + st * a.n_blk32;
    constexpr int PIECES = sizeof(Block) / 16, PER = (PIECES + 255) / 256;
    static_assert(sizeof(Block) % 16 == 0, "blocks move in 16-byte pieces");
    u32x4 next[PER];
    auto fetch = [&](int it) __attribute__((always_inline)) {
        const int b = min(first + 2 * it + grp, a.n_blk32 - 1);
        const u32x4 *p = reinterpret_cast<const u32x4 *>(src + b);
#pragma unroll
        for (int i = 0; i < PER; i++) next[i] = p[min((tid & 255) + 256 * i, PIECES - 1)];
    };
    auto stage = [&](int it) __attribute__((always_inline)) {
        u32x4 *p = reinterpret_cast<u32x4 *>(buf + 2 * grp + (it & 1));
#pragma unroll
        for (int i = 0; i < PER; i++)
            if ((tid & 255) + 256 * i < PIECES) p[(tid & 255) + 256 * i] = next[i];
    };
    fetch(0);
    // this wave's keys: row j of tile i is key base + 32 i + j
    half8 ka[NT][NKS];
    int6v k6[NT][NG];
    float sk[NT][16];
    {
        const DeqConstV dk;
        const uint32_t *kw = reinterpret_cast<const uint32_t *>(a.L.kp + st * a.L.P * (HD / 2));
        const float *ks = a.L.ks + st * a.L.P;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int p = min(base + 32 * i + j, a.L.P - 1);
#pragma unroll
            for (int t = 0; t < NKS; t++) ka[i][t] = dequant8_c(kw[k_word_idx<HD>(p, 2 * t + hf)], dk);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const half8 x[4] = {ka[i][4 * g], ka[i][4 * g + 1], ka[i][4 * g + 2], ka[i][4 * g + 3]};
                k6[i][g] = fp6_of(x, 1.0f);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) sk[i][e] = ks[min(base + 32 * i + 8 * (e >> 2) + 4 * hf + (e & 3), a.L.P - 1)];
        }
    }
    float acc[NT][16];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][e] = 0.0f;
    stage(0);
    if (n_it > 1) fetch(1);
    __syncthreads();
    for (int it = 0; it < n_it; it++) {
        const Block &b = buf[2 * grp + (it & 1)];
        if (it + 1 < n_it) stage(it + 1);
        if (it + 2 < n_it) fetch(it + 2);
        const int cb = first + 2 * it + grp;
        if (cb < a.n_blk32) {
            floatx16 sc[NT];
#pragma unroll
            for (int i = 0; i < NT; i++) sc[i] = (floatx16)0.0f;
#pragma unroll
            for (int t = 0; t < NKS; t++) {
                const half8 q = b.hi[t][lane];
#pragma unroll
                for (int i = 0; i < NT; i++) sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[i][t], q, sc[i], 0, 0, 0);
            }
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    int6v q;
#pragma unroll
                    for (int e = 0; e < 3; e++) {
                        const uint64_t x = b.lo[g][u][e][lane];
                        q[2 * e] = (int)(uint32_t)x;
                        q[2 * e + 1] = (int)(x >> 32);
                    }
#pragma unroll
                    for (int i = 0; i < NT; i++) sc[i] = mfma_lo6(k6[i][g], q, sc[i], u ? kQlo2E8 : kQlo1E8);
                }
            const float back = b.back[j], lse = b.lse[j];
            const int c = kColBlk * cb + j;
            const int qpos = c < n_cols ? len + c / a.G : -1;  // the last slot the column sees
            // (uniform: some column of the block does not see some key of the wave)
            const bool mask = base + KEYS / 4 - 1 > len + kColBlk * cb / a.G || kColBlk * (cb + 1) > n_cols;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    float x = sc[i][e] * sk[i][e];
                    if constexpr (SOFTCAP) {
                        x = tanhf(x * back / a.softcap) * a.softcap * kLog2e - lse;
                    } else {
                        x = __builtin_fmaf(x, back, -lse);
                    }
                    sc[i][e] = __builtin_amdgcn_exp2f(x);
                }
            if (mask) {
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (base + 32 * i + 8 * (e >> 2) + 4 * hf + (e & 3) > qpos) sc[i][e] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][e] += sc[i][e];
        }
        __syncthreads();
    }
    // the sums of the 32 columns' lanes
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            float v = acc[i][e];
            v += dpp_f<0xB1>(v);
            v += dpp_f<0x4E>(v);
            v += dpp_f<0x141>(v);
            v += dpp_f<0x140>(v);
            auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            if (j == 0) part[grp][wk * (KEYS / 4) + 32 * i + 8 * (e >> 2) + 4 * hf + (e & 3)] = v;
        }
    __syncthreads();
    for (int x = tid; x < KEYS; x += 512) {
        const int p = key0 + x;
        if (p >= a.max_seq) break;
        const float v = part[0][x] + part[1][x];
        if (p < n)
            w[p] = a.fresh ? v : w[p] + v;
        else if (a.fresh)
            w[p] = 0.0f;
    }
}

uint64_t col_block_bytes(int hd) {
    return hd == 256 ? sizeof(ColBlock<256>) : hd == 128 ? sizeof(ColBlock<128>) : sizeof(ColBlock<64>);
}

uint64_t part_floats(int rows, int pieces, int hd) { return pieces > 1 ? (uint64_t)rows * pieces * (hd + 2) : (uint64_t)rows * 2; }

}  // namespace

uint64_t weigh_chunk_workspace(int n_seq, int n_tok, int n_head, int n_kv, int stored_hd, int max_seq, int n_cu) {
    const int G = n_head / n_kv, rows = n_seq * n_tok * n_head;
    // (a chain of a call whose longest sequence is short needs less than pieces do, one piece's sums alone)
    const uint64_t parts = part_floats(rows, own_pieces_cap(n_seq, n_tok, G, n_kv, max_seq, n_cu), stored_hd) * sizeof(float);
    const uint64_t blocks = (uint64_t)n_seq * n_kv * ((n_tok * G + kColBlk - 1) / kColBlk);
    return (parts + 15) / 16 * 16 + blocks * col_block_bytes(stored_hd);
}

hipError_t launch_weigh_chunk(const WeighCall &c, hipStream_t st) {
    const int G = c.n_head / c.L.H, rows = c.L.S * c.n_tok * c.n_head;
    SharedCall sc;
    sc.own = sc.pre = c.L;
    sc.prefix_seq = sc.prefix_len = 0;
    sc.d_len = c.d_len;
    sc.q = c.q;
    sc.n_head = c.n_head;
    sc.n_tok = c.n_tok;
    sc.rope = c.rope;
    sc.rope_pairs = c.rope_pairs;
    sc.rope_rows = c.rope_rows;
    sc.softcap = c.softcap;
    sc.out = c.out;
    sc.plan = own_plan(c.L.S, c.n_tok, G, c.L.H, c.own_max, c.n_cu);
    sc.part = reinterpret_cast<float *>(c.ws);
    sc.own_part = nullptr;
    sc.own_chunk = sc.own_split = 1;
    sc.hlen = -1;
    sc.k_new = sc.v_new = nullptr;
    sc.n_cu = c.n_cu;
    sc.stats = sc.part;
    const hipError_t e = launch_shared(sc, st);
    if (e != hipSuccess) return e;
    const uint64_t parts = part_floats(rows, sc.plan.own_pieces, c.L.hd) * sizeof(float);

    ChunkArgs a;
    a.L = c.L;
    a.len = c.d_len;
    a.q = c.q;
    a.rope = c.rope;
    a.rope_pairs = c.rope_pairs;
    a.rope_rows = c.rope_rows;
    a.n_head = c.n_head;
    a.G = G;
    a.n_tok = c.n_tok;
    a.n_blk32 = (c.n_tok * G + kColBlk - 1) / kColBlk;
    a.inv_sqrt_hd = 1.0f / sqrtf((float)c.L.hdr);
    a.softcap = c.softcap;
    a.slots = sc.plan.own_pieces;
    a.pm = sc.plan.chain ? sc.part : sc.part + (size_t)rows * a.slots * c.L.hd;
    a.pl = a.pm + (size_t)rows * a.slots;
    a.cols = c.ws + (parts + 15) / 16 * 16;
    a.max_seq = c.max_seq;
    a.w = c.w;
    a.fresh = c.fresh;
    const dim3 prep((a.n_blk32 + 3) / 4, c.L.H, c.L.S);
    const int slots = c.fresh || c.captured ? c.max_seq : c.own_max;
    const bool norm = c.L.qn != nullptr, pad = c.L.hdr != c.L.hd;
#define TS_COLS(HDV)                                                                                                     \
    {                                                                                                                    \
        constexpr size_t lp = (size_t)128 * (HDV + 4) * sizeof(float), lc = 4 * sizeof(ColBlock<HDV>);                     \
        static_assert(lc <= 156 * 1024 && lp <= 156 * 1024, "LDS of the column kernels");                                 \
        auto prep_k = norm ? (pad ? weigh_prep_kernel<HDV, true, true> : weigh_prep_kernel<HDV, true, false>)             \
                           : (pad ? weigh_prep_kernel<HDV, false, true> : weigh_prep_kernel<HDV, false, false>);          \
        auto cols_k = c.softcap > 0.0f ? weigh_cols_kernel<HDV, true> : weigh_cols_kernel<HDV, false>;                    \
        (void)hipFuncSetAttribute((const void *)prep_k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lp);             \
        (void)hipFuncSetAttribute((const void *)cols_k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lc);             \
        prep_k<<<prep, 256, lp, st>>>(a);                                                                                 \
        const dim3 grid((unsigned)((slots + kColKeys<HDV> - 1) / kColKeys<HDV> * c.L.H), c.L.S);                          \
        cols_k<<<grid, 512, lc, st>>>(a);                                                                                 \
    }
    if (c.L.hd == 256) TS_COLS(256)
    else if (c.L.hd == 128) TS_COLS(128)
    else TS_COLS(64)
#undef TS_COLS
    return hipGetLastError();
}

}  // namespace ts
