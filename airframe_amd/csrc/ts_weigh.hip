// ts_weigh.hip -- what every cached slot receives of the attention of new tokens, for gfx950.
//
// For the new tokens t and query heads h of one kv head, P[t,h,p] = softmax over the slots p the token
// sees: w[p] = (w[p]) + sum over t and h of P[t,h,p].  The sums over columns need each softmax's final
// reference and sum, so they come behind the attention itself (one token: ts_weigh_token.hip).
//
// A chunk: the attention itself is the window walk of ts_shared.hip over the own keys.  It leaves its columns' rotated q
// in the operand layout of the matrix cores, and every column's log2 sum lse, its own or (of pieces of the keys)
// the join's.  Then the scores are computed a second time with the keys held in registers and the columns streaming
// past, so that a slot's sum stays in its lane: w[p] += sum over the columns of 2^(x - lse).  The products are the walk's
// (q in f16 and two fp6 terms, the codes exact in f16), so P here is what the output was made of but for its rounding.
//   4 sequences of 1024-1536 slots, 512 tokens, 32 heads over 8 of 128 dims: walk 127 us, sums 67 (26 GFLOP of
// scores, 0.39 PFLOP/s; the low terms double the products; under the profiler, the call itself takes 175). Of its 159K cycles a
// SIMD 40K go to the matrix cores and 50K to the exponentials and their sums, the rest to the waits between them: two waves a
// SIMD is what the keys' registers allow.
//   32 tokens of 4 sequences of 1003-8003 slots: walk 35 us, join 8.5, sums 17 (the call 55); 64 tokens behind 32704 slots 72,
// 8.2 and 31 (103).
// (The sums' launch joining the pieces itself: 43 us and 41.5 before or behind its tiles, the two launches 41.4.)
#include <cfloat>

#include "ts_columns.h"
#include "ts_evict.h"
#include "ts_shared.h"

namespace ts {
namespace {

struct ChunkArgs {
    KvLayerView L;
    const int32_t *len;
    int n_head, G, n_tok, n_blk32;
    float softcap, inv_softcap;
    const float *part;  // of pieces: [rows][slots][HD], references and sums [rows][slots]
    int slots, own_chunk;
    float *out;
    void *cols;  // [S][H][n_blk32] ColBlock
    int max_seq;
    float *w;
    bool fresh;
    int tiles;  // weigh_window_kernel: tiles of keys per workgroup
};

// The join of one (token, head) row's pieces by a wave, lane l holding HD / 64 dims: the output, and the row's lse into its
// column.  Bound by the partials' round trips, eight pieces' loads together (34 MB of 4096 rows 8.4 us).
template <int HD>
__global__ __launch_bounds__(256) void weigh_join_kernel(ChunkArgs a) {
    constexpr int D = HD / 64;
    const int lane = threadIdx.x & 63, H = a.L.H, G = a.G;
    // (rows of one kv head on the XCD that wrote their parts)
    const int h = blockIdx.x % H, u = blockIdx.x / H * 4 + (threadIdx.x >> 6), rows = a.L.S * a.n_tok * a.n_head;
    if (u >= rows / H) return;
    const int t = u / G, g = u - t * G, s = t / a.n_tok, tok = t - s * a.n_tok, row = t * a.n_head + h * G + g;
    const int n = min((min(a.len[s] + a.n_tok, a.L.P) + a.own_chunk - 1) / a.own_chunk, a.slots);
    const float *po = a.part + (size_t)row * a.slots * HD, *pm = a.part + (size_t)rows * a.slots * HD + (size_t)row * a.slots;
    const float *pl = pm + (size_t)rows * a.slots;
    float M = kMinit;
    for (int i = lane; i < n; i += 64) M = fmaxf(M, pm[i]);
    M = wave_max(M);
    float acc[D] = {}, l = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 8) {
        float x[8][D], m[8], ls[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = min(i0 + k, n - 1);
#pragma unroll
            for (int e = 0; e < D; e++) x[k][e] = po[(size_t)i * HD + D * lane + e];
            m[k] = pm[i];
            ls[k] = pl[i];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i0 + k >= n) break;
            if (ls[k] == 0.0f) continue;  // (a piece without keys has no output; one of a NaN q has)
            const float e2 = __builtin_amdgcn_exp2f(m[k] - M);
#pragma unroll
            for (int e = 0; e < D; e++) acc[e] += e2 * x[k][e];
            l += e2 * ls[k];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float *o = a.out + (size_t)row * a.L.hdr;
#pragma unroll
    for (int e = 0; e < D; e++)
        if (D * lane + e < a.L.hdr) o[D * lane + e] = acc[e] * inv;
    const int c = tok * G + g;
    if (lane == 0)
        static_cast<ColBlock<HD> *>(a.cols)[((size_t)s * H + h) * a.n_blk32 + c / kColBlk].lse[c % kColBlk] = M + __log2f(l);
}

// A wave's tile: NT x 32 keys as the matrix cores' first operand (row j of part i is key 32 i + j), the codes in f16 and fp6.
template <int HD>
struct KeyTile {
    static constexpr int NT = HD > 128 ? 1 : 2, KEYS = 32 * NT, NKS = HD / 16, NG = NKS / 4;
    static constexpr int V = HD / 32 < 4 ? HD / 32 : 4, NV = HD / 32 / V;  // words of a slot and lane group, in vectors
    typedef uint32_t vec __attribute__((ext_vector_type(V)));
    typedef half8 F16[NT][NKS];
    typedef int6v F6[NT][NG];
    typedef vec Raw[NT][4][NV];
};

// Slots base .. of one stream (past P: slot P - 1).
template <int HD>
__device__ __forceinline__ void fetch_keys(typename KeyTile<HD>::Raw &r, const uint32_t *kw, int P, int base, int j) {
    using T = KeyTile<HD>;
#pragma unroll
    for (int i = 0; i < T::NT; i++) {
        const int p = min(base + 32 * i + j, P - 1);
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int c = 0; c < T::NV; c++)
                r[i][g][c] = *reinterpret_cast<const typename T::vec *>(kw + k_word_idx<HD>(p, 16 * c + 2 * g));
    }
}

// k-step t takes word 2 t + hf of the slot: lane group t % 4, word 2 (t / 4) + hf of its words.
template <int HD>
__device__ __forceinline__ void set_keys(const typename KeyTile<HD>::Raw &r, typename KeyTile<HD>::F16 &ka,
                                         typename KeyTile<HD>::F6 &k6, int hf, const DeqConst &dk) {
    using T = KeyTile<HD>;
#pragma unroll
    for (int i = 0; i < T::NT; i++) {
#pragma unroll
        for (int g = 0; g < T::NG; g++) {
            // (the fp6 operand element by element: as a copy of four half8 the compiler keeps all of ka in memory)
            half32 all;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int t = 4 * g + u, at = 2 * g % T::V;
                const typename T::vec v = r[i][u][2 * g / T::V];
                const uint32_t w0 = v[at], w1 = v[at + 1];
                const half8 x = dequant8_c(hf ? w1 : w0, dk);
                ka[i][t] = x;
#pragma unroll
                for (int e = 0; e < 8; e++) all[8 * u + e] = x[e];
            }
            k6[i][g] = __builtin_amdgcn_cvt_scalef32_pk32_fp6_f16(all, 1.0f);
        }
    }
    // (pinned: the compiler would otherwise keep the codes and unpack them for every column block)
#pragma unroll
    for (int i = 0; i < T::NT; i++) {
#pragma unroll
        for (int t = 0; t < T::NKS; t++) {
            u32x4 x = __builtin_bit_cast(u32x4, ka[i][t]);
            asm volatile("" : "+v"(x));
            ka[i][t] = __builtin_bit_cast(half8, x);
        }
#pragma unroll
        for (int g = 0; g < T::NG; g++) asm volatile("" : "+v"(k6[i][g]));
    }
}

// Scores of one column block: lane (j, hf) holds column j and keys 32 i + 8 (e / 4) + 4 hf + e % 4.  Products are summed in
// the walk's order, so that a score has the same bits in both passes.
template <int HD>
__device__ __forceinline__ void tile_scores(const typename KeyTile<HD>::F16 &ka, const typename KeyTile<HD>::F6 &k6,
                                            const ColBlock<HD> &b, int lane, floatx16 (&sc)[KeyTile<HD>::NT]) {
    using T = KeyTile<HD>;
#pragma unroll
    for (int i = 0; i < T::NT; i++) sc[i] = (floatx16)0.0f;
#pragma unroll
    for (int g = 0; g < T::NG; g++) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const half8 q = b.hi[4 * g + u][lane];
#pragma unroll
            for (int i = 0; i < T::NT; i++) sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[i][4 * g + u], q, sc[i], 0, 0, 0);
        }
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
            for (int i = 0; i < T::NT; i++) sc[i] = mfma_lo6(k6[i][g], q, sc[i], u ? kQlo2E8 : kQlo1E8);
        }
    }
    // the columns' reads (one for an f16 step, three for a low term) run at least three ahead of the matrix instructions
    // that take them: four, then two behind each f16 step and one behind each low term
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int k = 0; k < 6 * T::NG; k++) {
        __builtin_amdgcn_sched_group_barrier(0x8, T::NT, 0);
        if (k >= 6 * T::NG - 3) continue;  // (all are out)
        if (k % 6 < 4) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// Probabilities of one column block added to acc.  sk: the tile's K scales times kSkUnit, in LDS; cb: the block, of n_cols columns in
// all; base: the tile's first key.
template <int HD, bool SOFTCAP>
__device__ __forceinline__ void add_probs(floatx16 (&sc)[KeyTile<HD>::NT], float (&acc)[KeyTile<HD>::NT][16], const ColBlock<HD> &b,
                                          const float *sk, int cb, int n_cols, int G, int len, int base, int j, int hf,
                                          float softcap, float inv_softcap) {
    constexpr int NT = KeyTile<HD>::NT;
    const float back = b.back[j], lse = b.lse[j];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const floatx4 s4 = *reinterpret_cast<const floatx4 *>(sk + 32 * i + 8 * q + 4 * hf);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                // (the walk's bits: window_scores_again)
                const float t = sc[i][4 * q + r] * s4[r];
                float x;
                if constexpr (SOFTCAP) x = cap<true>(t * back, softcap, inv_softcap) - lse;
                else x = __builtin_fmaf(t, back, -lse);
                sc[i][4 * q + r] = __builtin_amdgcn_exp2f(x);
            }
        }
    // (uniform: some column of the block does not see some key of the tile)
    if (base + 32 * NT - 1 > len + kColBlk * cb / G || kColBlk * (cb + 1) > n_cols) {
        asm volatile("");  // (a branch: the compares are the rare case)
        const int c = kColBlk * cb + j;
        const int qpos = c < n_cols ? len + c / G : -1;  // the last slot the column sees
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

// The sums over the 32 columns' lanes into the tile's row of LDS.
template <int HD>
__device__ __forceinline__ void sum_columns(const float (&acc)[KeyTile<HD>::NT][16], float *row, int j, int hf) {
#pragma unroll
    for (int i = 0; i < KeyTile<HD>::NT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            float v = acc[i][e];
            v += dpp_f<0xB1>(v);
            v += dpp_f<0x4E>(v);
            v += dpp_f<0x141>(v);
            v += dpp_f<0x140>(v);
            auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            if (j == 0) row[32 * i + 8 * (e >> 2) + 4 * hf + (e & 3)] = v;
        }
}

constexpr int kWaves = 8;  // of a workgroup

// Few columns: all of them in LDS, and every wave takes tiles of keys of its own, the next one's codes on their way.
// No barrier but the one behind the columns.  Grid: kv head first, so that the workgroups that read one head's
// columns share an XCD where the heads divide the XCDs; sequences last (before the tiles a ragged batch of four took 27.6 us
// instead of 18.4: its longest sequence's workgroups, every fourth, meet on the same CUs).  Bound by its chain: the columns and the first codes from L2
// and HBM, then tile by tile the two passes' products without a neighbour (150 KB of columns leave one workgroup a CU).
template <int HD, bool SOFTCAP>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_window_kernel(ChunkArgs a) {
    using Tile = KeyTile<HD>;
    using Block = ColBlock<HD>;
    constexpr int NT = Tile::NT, KEYS = Tile::KEYS;
    extern __shared__ __align__(16) unsigned char win_smem[];
    Block *const blk = reinterpret_cast<Block *>(win_smem);  // [n_blk32]
    __shared__ __align__(16) float sks[kWaves][KEYS], sums[kWaves][KEYS];
    const int H = a.L.H, h = blockIdx.x % H, s = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t st = (size_t)s * H + h;
    const int len = a.len[s], n = len + a.n_tok, n_cols = a.n_tok * a.G;
    const int first = blockIdx.x / H * a.tiles, last = first + a.tiles;
    float *const w = a.w + st * a.max_seq;
    if (n > a.max_seq) return;  // (a graph replayed past the capacity)
    const float *ks = a.L.ks + st * a.L.P;
    const uint32_t *const kw = reinterpret_cast<const uint32_t *>(a.L.kp + st * a.L.P * (HD / 2));
    typename Tile::Raw raw;
    float scale = 0.0f;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        fetch_keys<HD>(raw, kw, a.L.P, tile * KEYS, j);
        scale = ks[min(tile * KEYS + (lane & (KEYS - 1)), a.L.P - 1)] * kSkUnit;
    };
    if (first * KEYS < n) {
        fetch(min(first + wave, (n - 1) / KEYS));
        const u32x4 *src = reinterpret_cast<const u32x4 *>(static_cast<const Block *>(a.cols) + st * a.n_blk32);
        u32x4 *to = reinterpret_cast<u32x4 *>(blk);
        const int pieces = a.n_blk32 * (int)(sizeof(Block) / 16);
#pragma unroll 4
        for (int i = tid; i < pieces; i += 64 * kWaves) to[i] = src[i];
    }
    __syncthreads();
    const DeqConstV dk;
    for (int tile = first + wave; tile < last; tile += kWaves) {
        const int base = tile * KEYS, p = base + lane;
        if (base >= a.max_seq) break;
        const bool mine = lane < KEYS && p < a.max_seq;
        if (base >= n) {
            if (a.fresh && mine) w[p] = 0.0f;
            continue;
        }
        const float old = !a.fresh && mine && p < n ? w[p] : 0.0f;
        typename Tile::F16 ka;
        typename Tile::F6 k6;
        set_keys<HD>(raw, ka, k6, hf, dk);
        sks[wave][lane & (KEYS - 1)] = scale;
        fetch(min(tile + kWaves, (n - 1) / KEYS));
        asm volatile("" ::: "memory");
        float acc[NT][16];
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][e] = 0.0f;
        // (the first columns that see a key of the tile; all blocks behind them do too)
        for (int cb = max(0, base - len) * a.G / kColBlk; cb < a.n_blk32; cb++) {
            floatx16 sc[NT];
            tile_scores<HD>(ka, k6, blk[cb], lane, sc);
            add_probs<HD, SOFTCAP>(sc, acc, blk[cb], sks[wave], cb, n_cols, a.G, len, base, j, hf, a.softcap, a.inv_softcap);
        }
        sum_columns<HD>(acc, sums[wave], j, hf);
        asm volatile("" ::: "memory");  // (the wave's LDS writes are ordered before its reads)
        if (mine) {
            const float v = sums[wave][lane & (KEYS - 1)];
            if (p < n) w[p] = old + v;
            else if (a.fresh) w[p] = 0.0f;
        }
    }
}

// Many columns: KW waves hold KW tiles of keys for as long as the columns stream past through LDS; the workgroup's
// groups of KW waves take the column blocks in turn.  (Two groups half a step apart, one's matrix instructions
// beside the other's exponentials: 70 us, 68 without, 512 tokens of 4 sequences of 1-1.5K slots.)
template <int HD, bool SOFTCAP, int KW>
__global__ __launch_bounds__(64 * kWaves, 2) void weigh_cols_kernel(ChunkArgs a) {
    using Tile = KeyTile<HD>;
    using Block = ColBlock<HD>;
    constexpr int NT = Tile::NT, TK = Tile::KEYS, KEYS = KW * TK, GROUPS = kWaves / KW, GT = 64 * KW;
    extern __shared__ __align__(16) unsigned char cols_smem[];
    Block *const buf = reinterpret_cast<Block *>(cols_smem);  // [group][2]
    __shared__ __align__(16) float part[GROUPS][KEYS], sks[KEYS];
    const int H = a.L.H, h = blockIdx.x % H, kb = blockIdx.x / H, s = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = wave / KW, wk = wave % KW, gt = tid % GT;
    const size_t st = (size_t)s * H + h;
    const int len = a.len[s], n = len + a.n_tok, key0 = kb * KEYS;
    float *const w = a.w + st * a.max_seq;
    if (n > a.max_seq) return;  // (a graph replayed past the capacity)
    if (key0 >= n) {
        if (a.fresh)
            for (int p = key0 + tid; p < min(key0 + KEYS, a.max_seq); p += 64 * kWaves) w[p] = 0.0f;
        return;
    }
    const int base = key0 + wk * TK, n_cols = a.n_tok * a.G;
    // (the first columns that see a key of the block; all blocks behind them do too)
    const int first = max(0, key0 - len) * a.G / kColBlk;
    const int n_it = (a.n_blk32 - first + GROUPS - 1) / GROUPS;
    const Block *const src = static_cast<const Block *>(a.cols) + st * a.n_blk32;
    constexpr int PIECES = sizeof(Block) / 16, PER = (PIECES + GT - 1) / GT;
    static_assert(sizeof(Block) % 16 == 0, "blocks move in 16-byte pieces");
    u32x4 next[PER];
    auto fetch = [&](int it) __attribute__((always_inline)) {
        const int b = min(first + GROUPS * it + grp, a.n_blk32 - 1);
        const u32x4 *p = reinterpret_cast<const u32x4 *>(src + b);
#pragma unroll
        for (int i = 0; i < PER; i++) next[i] = p[min(gt + GT * i, PIECES - 1)];
    };
    auto stage = [&](int it) __attribute__((always_inline)) {
        u32x4 *p = reinterpret_cast<u32x4 *>(buf + 2 * grp + (it & 1));
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (gt + GT * i < PIECES) p[gt + GT * i] = next[i];
    };
    fetch(0);
    typename Tile::F16 ka;
    typename Tile::F6 k6;
    {
        const DeqConstV dk;
        typename Tile::Raw raw;
        fetch_keys<HD>(raw, reinterpret_cast<const uint32_t *>(a.L.kp + st * a.L.P * (HD / 2)), a.L.P, base, j);
        if (tid < KEYS) sks[tid] = a.L.ks[st * a.L.P + min(key0 + tid, a.L.P - 1)] * kSkUnit;
        set_keys<HD>(raw, ka, k6, hf, dk);
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
        const int cb = first + GROUPS * it + grp;
        floatx16 sc[NT];
        tile_scores<HD>(ka, k6, b, lane, sc);
        if (it + 1 < n_it) stage(it + 1);
        if (it + 2 < n_it) fetch(it + 2);
        // (a block behind the last has no columns: nothing is added)
        add_probs<HD, SOFTCAP>(sc, acc, b, sks + wk * TK, cb, n_cols, a.G, len, base, j, hf, a.softcap, a.inv_softcap);
        __syncthreads();
    }
    sum_columns<HD>(acc, part[grp] + wk * TK, j, hf);
    __syncthreads();
    for (int x = tid; x < KEYS; x += 64 * kWaves) {
        const int p = key0 + x;
        if (p >= a.max_seq) break;
        float v = part[0][x];
#pragma unroll
        for (int i = 1; i < GROUPS; i++) v += part[i][x];
        if (p < n)
            w[p] = a.fresh ? v : w[p] + v;
        else if (a.fresh)
            w[p] = 0.0f;
    }
}

size_t col_block_bytes(int hd) {
    return hd == 256 ? sizeof(ColBlock<256>) : hd == 128 ? sizeof(ColBlock<128>) : sizeof(ColBlock<64>);
}

uint64_t part_bytes(uint64_t rows, int pieces, int hd) { return pieces > 1 ? (rows * pieces * (hd + 2) * sizeof(float) + 15) / 16 * 16 : 0; }

// The columns' blocks and the waves' rows in a CU's LDS.
constexpr size_t kWindowLds = 150 * 1024;

}  // namespace

uint64_t weigh_chunk_workspace(int n_seq, int n_tok, int n_head, int n_kv, int stored_hd, int max_seq, int n_cu) {
    const int G = n_head / n_kv;
    const uint64_t blocks = (uint64_t)n_seq * n_kv * ((n_tok * G + kColBlk - 1) / kColBlk);
    return part_bytes((uint64_t)n_seq * n_tok * n_head, own_pieces_cap(n_seq, n_tok, G, n_kv, max_seq, n_cu), stored_hd) +
           blocks * col_block_bytes(stored_hd);
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
    sc.plan = own_plan(c.n_ctx, c.L.S, c.n_tok, G, c.L.H, c.n_cu);
    sc.part = reinterpret_cast<float *>(c.ws);
    sc.own_part = nullptr;
    sc.own_chunk = sc.own_split = 1;
    sc.hlen = -1;
    sc.k_new = sc.v_new = nullptr;
    sc.n_cu = c.n_cu;
    sc.cols = c.ws + part_bytes(rows, sc.plan.own_pieces, c.L.hd);
    sc.n_blk32 = (c.n_tok * G + kColBlk - 1) / kColBlk;
    const hipError_t e = launch_shared(sc, st);
    if (e != hipSuccess) return e;

    ChunkArgs a;
    a.L = c.L;
    a.len = c.d_len;
    a.n_head = c.n_head;
    a.G = G;
    a.n_tok = c.n_tok;
    a.n_blk32 = sc.n_blk32;
    a.softcap = c.softcap;
    a.inv_softcap = c.softcap > 0.0f ? std::min(1.0f / c.softcap, FLT_MAX) : 0.0f;
    a.part = sc.part;
    a.slots = sc.plan.own_pieces;
    a.own_chunk = sc.plan.own_chunk;
    a.out = c.out;
    a.cols = sc.cols;
    a.max_seq = c.max_seq;
    a.w = c.w;
    a.fresh = c.fresh;
    const int slots = c.fresh || c.captured ? c.max_seq : c.own_max;
    const bool window = a.n_blk32 * col_block_bytes(c.L.hd) <= kWindowLds;
    // Few columns: tiles of keys per workgroup, one for every wave at least and a workgroup per CU over the batch's keys;
    // where that leaves CUs idle, one for every second wave (11 sequences of 4-726 slots, 37 tokens of 64 heads with
    // softcap: 44 us with eight tiles, 32 with four).
    const int tk = c.L.hd > 128 ? 32 : 64;
    int64_t tiles = 0, wg4 = 0, wg2 = 0;
    for (int s = 0; s < c.L.S; s++) {
        tiles += (c.n_ctx[s] + tk - 1) / tk * c.L.H;
        wg4 += (c.n_ctx[s] + 4 * tk - 1) / (4 * tk) * c.L.H;
        wg2 += (c.n_ctx[s] + 2 * tk - 1) / (2 * tk) * c.L.H;
    }
    const int64_t per_cu = (tiles + c.n_cu - 1) / c.n_cu;
    a.tiles = (int)(per_cu <= kWaves / 2 ? kWaves / 2 : (per_cu + kWaves - 1) / kWaves * kWaves);
    // Many columns: four tiles of keys per workgroup, or two, whose column groups then have half as many steps, if that
    // takes less than twice as many rounds of the CUs.  4 sequences of 434 slots, 505 tokens, 64-dim heads with softcap:
    // 112 and 63 us (the launch).
    const bool two = 2 * ((wg4 + c.n_cu - 1) / c.n_cu) > (wg2 + c.n_cu - 1) / c.n_cu && c.L.hd <= 128;
#define TS_COLS(HDV)                                                                                                     \
    {                                                                                                                    \
        if (!sc.plan.chain) weigh_join_kernel<HDV><<<(unsigned)((rows / c.L.H + 3) / 4 * c.L.H), 256, 0, st>>>(a);         \
        constexpr int TK = KeyTile<HDV>::KEYS, KW2 = HDV <= 128 ? 2 : 4;                                                 \
        const bool cap = c.softcap > 0.0f;                                                                               \
        auto kernel = window ? (cap ? weigh_window_kernel<HDV, true> : weigh_window_kernel<HDV, false>)                   \
                      : two  ? (cap ? weigh_cols_kernel<HDV, true, KW2> : weigh_cols_kernel<HDV, false, KW2>)             \
                             : (cap ? weigh_cols_kernel<HDV, true, 4> : weigh_cols_kernel<HDV, false, 4>);                \
        const int kw = two ? KW2 : 4, per = TK * (window ? a.tiles : kw);                                                \
        const int lds = (int)sizeof(ColBlock<HDV>) * (window ? a.n_blk32 : 2 * kWaves / kw);                             \
        static_assert(sizeof(ColBlock<HDV>) * 2 * kWaves / KW2 <= kWindowLds, "the column groups' blocks fit a CU's LDS"); \
        (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,                       \
                                  window ? (int)kWindowLds : lds);                                                       \
        kernel<<<dim3((unsigned)((slots + per - 1) / per * c.L.H), c.L.S), 64 * kWaves, lds, st>>>(a);                    \
    }
    if (c.L.hd == 256) TS_COLS(256)
    else if (c.L.hd == 128) TS_COLS(128)
    else TS_COLS(64)
#undef TS_COLS
    return hipGetLastError();
}

}  // namespace ts
