// ts_packed.hip -- rotary positions, and the INT4 cache written from and read into packed rows,
// for gfx950.
//
// All of these move bytes: a few operations per element, so what bounds them is HBM, and at a few
// rows the launch.  Their arithmetic rounds like the CPU quantizer (one rounding per operation,
// no contraction), which is what makes codes and scales those of the other append entry points.
#include "ts_packed.h"
#include "ts_store.h"

namespace ts {
namespace {

// ---- rotary positions ---------------------------------------------------------------------------

// Entry (p, i) = mult (cos, sin)(p theta_i), the angle in 64 bits: in 32 the product p theta_i alone
// is off by up to 2^-24 p radians, 0.008 at 131072.  theta_i = base^(-2i / rope_dim) scaled by parts:
// r = l_train theta_i / 2 pi turns fit the trained length; ramp = clamp((r - alpha) / (beta - alpha)),
// theta_i ((1 - ramp) / factor + ramp); without beta > alpha all are divided by factor.  Once per table: 14 us
// for 40960 positions of 48 pairs.
__global__ __launch_bounds__(256) void rope_table_kernel(float2 *table, int n_pos, int pairs, double base, double factor,
                                                         double l_train, double alpha, double beta, double mult) {
    const int i = blockIdx.x * 64 + (threadIdx.x & 63);
    if (i >= pairs) return;
    double theta = pow(base, -2.0 * i / (2.0 * pairs));
    if (beta > alpha) {
        const double r = (l_train * theta / 6.283185307179586476925 - alpha) / (beta - alpha);
        const double ramp = fmin(fmax(r, 0.0), 1.0);
        theta = theta * ((1.0 - ramp) / factor + ramp);
    } else {
        theta = theta / factor;
    }
    for (int p = blockIdx.y * 4 + (threadIdx.x >> 6); p < n_pos; p += gridDim.y * 4) {
        double s, c;
        sincos(p * theta, &s, &c);
        table[(size_t)p * pairs + i] = make_float2((float)(c * mult), (float)(s * mult));
    }
}

struct RopeArgs {
    const void *x;
    void *out;
    int64_t xs, os;  // elements from one token's row to the next
    const int32_t *pos;
    const float2 *table;
    int n_tok, n_head, hd, pairs, n_pos;
    int units, rot_units;  // work items per head row, and those of them that rotate
    int groups;            // of HPT heads
    bool in_place;
};

enum { kInterleaved = 0, kHalf = 1, kHalfOdd = 2 };

// The rotations of pairs u0 .. u0 + N - 1 at position p: identity past the rotated pairs, NaN for a
// position that the table does not have (there is no value for such a row, and it must not
// pass for one).
template <int N>
__device__ inline void rotations(const RopeArgs &a, int p, int u0, float2 (&cs)[N]) {
    const bool ok = p >= 0 && p < a.n_pos;
    const float2 *row = a.table + (size_t)(ok ? p : 0) * a.pairs;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float2 t = row[min(u0 + i, a.pairs - 1)];
        cs[i] = u0 + i >= a.pairs ? make_float2(1.0f, 0.0f) : ok ? t : make_float2(NAN, NAN);
    }
}

// One work item of HPT heads of one token: 8 consecutive dims (interleaved pairs), 8 dims of each
// half of the rotated part, or 8 dims behind it; a single pair or dim where the halves are no
// multiple of 8.  A thread keeps its rotations for its HPT heads, so that the table's rows (8
// bytes a pair) are read once for HPT rows of x.
// HBM: 14.8k tokens of 32 bf16 heads (249 MB read and written) in 37.8 us, 6.6 TB/s (part of it still in
// the last-level cache); 32 tokens of 40 heads 3.1 us, which is a launch.
template <class T, int LAYOUT, int HPT>
__global__ __launch_bounds__(256) void rope_apply_kernel(RopeArgs a) {
    const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
    const uint32_t per_tok = a.units * a.groups;
    const uint32_t tok = idx / per_tok;
    if (tok >= (uint32_t)a.n_tok) return;
    const uint32_t rest = idx - tok * per_tok;
    const int g = rest / a.units, u = rest - g * a.units;
    const bool turns = u < a.rot_units;
    if (!turns && a.in_place) return;
    const int p = a.pos[tok];
    const T *x = static_cast<const T *>(a.x) + (int64_t)tok * a.xs;
    T *out = static_cast<T *>(a.out) + (int64_t)tok * a.os;
    if constexpr (LAYOUT == kHalfOdd) {
        float2 cs[1];
        rotations<1>(a, p, turns ? u : 0, cs);
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int h = g * HPT + i;
            if (h >= a.n_head) break;
            const size_t at = (size_t)h * a.hd;
            if (turns) {
                float v0 = (float)x[at + u], v1 = (float)x[at + a.pairs + u];
                rope_rotate(v0, v1, cs[0]);
                out[at + u] = (T)v0;
                out[at + a.pairs + u] = (T)v1;
            } else {
                out[at + a.pairs + u] = x[at + a.pairs + u];
            }
        }
    } else if constexpr (LAYOUT == kHalf) {
        float2 cs[8];
        if (turns) rotations<8>(a, p, 8 * u, cs);
        float v0[HPT][8], v1[HPT][8];
        const int d0 = turns ? 8 * u : 8 * u + a.pairs;  // (rot_units = pairs / 8)
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int h = min(g * HPT + i, a.n_head - 1);
            load8(x + (size_t)h * a.hd + d0, v0[i]);
            if (turns) load8(x + (size_t)h * a.hd + d0 + a.pairs, v1[i]);
        }
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int h = g * HPT + i;
            if (h >= a.n_head) break;
            if (turns) {
#pragma unroll
                for (int e = 0; e < 8; e++) rope_rotate(v0[i][e], v1[i][e], cs[e]);
                store8(out + (size_t)h * a.hd + d0 + a.pairs, v1[i]);
            }
            store8(out + (size_t)h * a.hd + d0, v0[i]);
        }
    } else {
        float2 cs[4];
        if (turns) rotations<4>(a, p, 4 * u, cs);
        float v[HPT][8];
#pragma unroll
        for (int i = 0; i < HPT; i++) load8(x + (size_t)min(g * HPT + i, a.n_head - 1) * a.hd + 8 * u, v[i]);
#pragma unroll
        for (int i = 0; i < HPT; i++) {
            const int h = g * HPT + i;
            if (h >= a.n_head) break;
            if (turns) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * u + e < a.pairs) rope_rotate(v[i][2 * e], v[i][2 * e + 1], cs[e]);
            }
            store8(out + (size_t)h * a.hd + 8 * u, v[i]);
        }
    }
}

template <class T, int HPT>
hipError_t rope_apply_typed(RopeArgs a, int layout, hipStream_t st) {
    a.groups = (a.n_head + HPT - 1) / HPT;
    const int64_t per_tok = (int64_t)a.units * a.groups;
    const int64_t most = std::max<int64_t>(1, (int64_t)0x7FFFFF00 / per_tok);  // tokens that 31 bits of items hold
    const int n_tok = a.n_tok;
    for (int64_t t0 = 0; t0 < n_tok; t0 += most) {
        RopeArgs b = a;
        b.n_tok = (int)std::min<int64_t>(most, n_tok - t0);
        b.x = static_cast<const T *>(a.x) + t0 * a.xs;
        b.out = static_cast<T *>(a.out) + t0 * a.os;
        b.pos = a.pos + t0;
        const unsigned blocks = (unsigned)((b.n_tok * per_tok + 255) / 256);
        if (layout == kInterleaved)
            rope_apply_kernel<T, kInterleaved, HPT><<<blocks, 256, 0, st>>>(b);
        else if (layout == kHalf)
            rope_apply_kernel<T, kHalf, HPT><<<blocks, 256, 0, st>>>(b);
        else
            rope_apply_kernel<T, kHalfOdd, HPT><<<blocks, 256, 0, st>>>(b);
    }
    return hipGetLastError();
}

// ---- the cache from packed rows -------------------------------------------------------------------

// Work items of n new rows: the 32-position blocks that they can touch, wherever they start.
inline int append_items(int n) { return n > 0 ? (n + 30) / kBlk + 1 : 0; }

// One workgroup writes the new positions of one 32-position block of one (sequence, kv head), as the
// append kernels of equal-length rows do (store_block64 / 128 / 256: it owns the block's V words,
// which interleave 8 positions).  Rows of any type are widened in registers.
// VALU work bounds it (rotation, maxima, codes that are the CPU's to the bit, V words put together), not HBM:
// 15.2k tokens of 8 f32 heads of 128 dims (125 + 17 MB) 28.5 us, 5.0 TB/s, in f16 (half the bytes) 28.1; 28k
// tokens of 8 bf16 heads of 80 dims (72 + 30 MB) 45.6 us, 2.2 TB/s: the 48 padded dims cost the same work
// as the others.  Eight waves per SIMD instead of six (64 registers) changed nothing for 16-bit rows, and
// f32 rows spilled.
template <class T, int HD>
__global__ __launch_bounds__(256) void append_packed_kernel(KvLayerView L, PackTable t, const int32_t *__restrict__ d_len,
                                                            const T *__restrict__ k, int64_t k_stride,
                                                            const T *__restrict__ v, int64_t v_stride,
                                                            const float *__restrict__ rope, int rope_pairs, int n_pos) {
    constexpr int LPR = HD / 8;        // lanes per position
    constexpr int NR = HD == 64 ? 1 : HD / 64;  // positions per lane
    const int item = blockIdx.x / L.H, h = blockIdx.x - item * L.H;
    const int i = pack_find(t, item), s = t.seq0 + i;
    const int row0 = t.tok[i], count = t.tok[i + 1] - row0;
    const int start = d_len[s];
    const int end = min(start + count, L.P);  // (a graph replayed past capacity writes nothing past it)
    const int blk = start / kBlk + (item - t.item[i]);
    const int p0 = blk * kBlk;
    if (p0 >= end) return;
    const int lo = max(p0, start), hi = min(p0 + kBlk, end);
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane / LPR, l = lane % LPR;
    const bool in = 8 * l < L.hdr;  // (lanes past the row load its first dims and drop them)
    float kx[NR][8], vx[NR][8];
    float2 cs[NR][4];
#pragma unroll
    for (int rd = 0; rd < NR; rd++) {
        const int at = HD == 64    ? 4 * wave + (r & 3) + 16 * (r >> 2)
                       : HD == 128 ? 16 * rd + 4 * wave + r
                                   : 4 * wave + 2 * (rd & 1) + r + 16 * (rd >> 1);
        const int pc = min(max(p0 + at, lo), hi - 1);  // (a position outside loads a neighbour's row)
        const int pr = min(rot_of(L, s, pc), n_pos - 1);
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const int pair = 4 * l + m;
            cs[rd][m] = pair < rope_pairs ? *reinterpret_cast<const float2 *>(rope + ((size_t)pr * rope_pairs + pair) * 2)
                                          : make_float2(1.0f, 0.0f);
        }
        const int64_t row = row0 + (pc - start);
        const int64_t at_h = (int64_t)h * L.hdr + 8 * (in ? l : 0);
        load8(k + row * k_stride + at_h, kx[rd]);
        load8(v + row * v_stride + at_h, vx[rd]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            kx[rd][e] = in ? kx[rd][e] : 0.0f;
            vx[rd][e] = in ? vx[rd][e] : 0.0f;
        }
    }
    if constexpr (HD == 64)
        store_block64<sizeof(T) == 2>(L, s, h, blk, lo, hi, kx[0], vx[0], cs[0], rope_pairs, wave, lane);
    else if constexpr (HD == 128)
        store_block128<sizeof(T) == 2>(L, s, h, blk, lo, hi, kx, vx, cs, rope_pairs, wave, lane);
    else
        store_block256<sizeof(T) == 2>(L, s, h, blk, lo, hi, kx, vx, cs, rope_pairs, wave, lane);
}

// ---- and back ---------------------------------------------------------------------------------------

// Work items of n positions from p0 on: the 32-position blocks that hold them.
inline int read_items(int p0, int n) { return n > 0 ? (p0 + n - 1) / kBlk - p0 / kBlk + 1 : 0; }

// (code - 8) scale of 8 codes, each rounded once to 32 bits.
__device__ inline void values8(uint32_t w, float scale, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)((int)((w >> (4 * e)) & 0xFu) - 8) * scale;
}

// One workgroup reads one 32-position block of one (sequence, kv head).  A thread writes 8 dims of one
// row: one K word, and one nibble each of 8 V words, which pass through LDS (a V word holds one dim
// of 8 positions).  HBM: 15.3k tokens of 8 f32 heads of 128 dims 26.9 us, 5.3 TB/s; 8 bf16 heads of 80
// dims of 28k tokens 19.5 us, 5.2 TB/s.
template <class T, int HD>
__global__ __launch_bounds__(256) void read_packed_kernel(KvLayerView L, PackTable t, T *__restrict__ k, int64_t k_stride,
                                                          T *__restrict__ v, int64_t v_stride) {
    __shared__ uint4 vw[HD];
    const int item = blockIdx.x / L.H, h = blockIdx.x - item * L.H;
    const int i = pack_find(t, item), s = t.seq0 + i;
    const int start = t.pos0[i], row0 = t.tok[i], end = start + t.tok[i + 1] - row0;
    const int blk = start / kBlk + (item - t.item[i]), p0 = blk * kBlk;
    const int tid = threadIdx.x;
    const size_t row = (size_t)s * L.H + h;
    const uint4 *vsrc = reinterpret_cast<const uint4 *>(L.vp + (row * (L.P / kBlk) + blk) * (HD * 16));
    for (int c = tid; c < HD; c += 256) vw[c] = vsrc[c];
    const uint32_t *kw = reinterpret_cast<const uint32_t *>(L.kp + row * L.P * (HD / 2));
    __syncthreads();
    const uint32_t *vb = reinterpret_cast<const uint32_t *>(vw);
    const int wpr = L.hdr / 8;
    constexpr int U = HD / 8;
#pragma unroll
    for (int c = tid; c < kBlk * U; c += 256) {
        const int q = c / U, u = c % U, p = p0 + q;
        if (p < start || p >= end || u >= wpr) continue;
        const int64_t dst = row0 + (p - start);
        float x[8];
        values8(kw[k_word_idx<HD>(p, u)], L.ks[row * L.P + p], x);
        store8(k + dst * k_stride + (int64_t)h * L.hdr + 8 * u, x);
        const int g = (q & 15) >> 2, n = (q & 3) + 4 * (q >> 4);
        const float sv = L.vs[row * L.P + p];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t w = vb[v_word_idx(g * 16 + 8 * (u & 1) + e, u >> 1)];
            x[e] = (float)((int)((w >> (4 * n)) & 0xFu) - 8) * sv;
        }
        store8(v + dst * v_stride + (int64_t)h * L.hdr + 8 * u, x);
    }
}

// Every length of the table's sequences grows by its rows.
__global__ __launch_bounds__(kPackSeqs) void len_add_kernel(int32_t *len, PackTable t) {
    const int i = threadIdx.x;
    if (i < t.n) len[t.seq0 + i] += t.tok[i + 1] - t.tok[i];
}

}  // namespace

hipError_t launch_rope_table(float *table, int32_t n_pos, int32_t rope_dim, double base, double factor, double l_train,
                             double alpha, double beta, double mult, hipStream_t st) {
    const int pairs = rope_dim / 2;
    const dim3 grid((pairs + 63) / 64, std::min((n_pos + 3) / 4, 2048));
    rope_table_kernel<<<grid, 256, 0, st>>>(reinterpret_cast<float2 *>(table), n_pos, pairs, base, factor, l_train, alpha,
                                            beta, mult);
    return hipGetLastError();
}

hipError_t launch_rope_apply(int32_t dtype, int32_t layout, const void *x, int64_t x_stride, const int32_t *pos, int n_tok,
                             int n_head, int hd, const float *table, int pairs, int n_pos, void *out, int64_t out_stride,
                             hipStream_t st) {
    RopeArgs a;
    a.x = x;
    a.out = out;
    a.xs = x_stride;
    a.os = out_stride;
    a.pos = pos;
    a.table = reinterpret_cast<const float2 *>(table);
    a.n_tok = n_tok;
    a.n_head = n_head;
    a.hd = hd;
    a.pairs = pairs;
    a.n_pos = n_pos;
    a.in_place = x == out;
    if (layout == TS_ROPE_INTERLEAVED) {
        a.units = hd / 8;
        a.rot_units = (pairs + 3) / 4;
    } else if (pairs % 8 == 0) {
        layout = kHalf;
        a.rot_units = pairs / 8;
        a.units = a.rot_units + (hd - 2 * pairs) / 8;
    } else {
        layout = kHalfOdd;
        a.rot_units = pairs;
        a.units = hd - pairs;
    }
    // Four heads to a thread once the items of 8 dims fill the chip, one each below.  16 bits, 32 + 8 heads of
    // 128 dims: 512 tokens 4.6 us with one head, 4.4 with four; 2048 tokens 10.6 and 8.5, 8192 31.5
    // and 27.9; 8 tokens 3.1 and 3.5, 128 tokens 3.4 and 3.7.  32 bits: 64 tokens (half layout) 3.6 and 4.3,
    // 2048 14.7 and 13.9, 8192 within 4% either way.
    const bool many = (int64_t)n_tok * n_head * a.units >= (1 << 18);
    if (dtype == TS_DTYPE_F32) return many ? rope_apply_typed<float, 4>(a, layout, st) : rope_apply_typed<float, 1>(a, layout, st);
    if (dtype == TS_DTYPE_F16)
        return many ? rope_apply_typed<_Float16, 4>(a, layout, st) : rope_apply_typed<_Float16, 1>(a, layout, st);
    return many ? rope_apply_typed<__bf16, 4>(a, layout, st) : rope_apply_typed<__bf16, 1>(a, layout, st);
}

#define TS_TYPED(LAUNCH)                                                        \
    {                                                                           \
        if (dtype == TS_DTYPE_F32) { using T = float; TS_HD(LAUNCH) }            \
        else if (dtype == TS_DTYPE_F16) { using T = _Float16; TS_HD(LAUNCH) }    \
        else { using T = __bf16; TS_HD(LAUNCH) }                                 \
    }
#define TS_HD(LAUNCH)                                              \
    {                                                              \
        if (L.hd == 64) { constexpr int HD = 64; LAUNCH; }          \
        else if (L.hd == 128) { constexpr int HD = 128; LAUNCH; }   \
        else { constexpr int HD = 256; LAUNCH; }                    \
    }

hipError_t launch_append_packed(const KvLayerView &L, const int32_t *d_len, int32_t dtype, const void *k, int64_t k_stride,
                                const void *v, int64_t v_stride, const int32_t *off, const float *rope, int32_t rope_pairs,
                                int32_t n_pos, hipStream_t st) {
    PackTable t;
    for (int s = 0; s < L.S; s += t.n) {
        pack_fill(t, off, nullptr, L.S, s, append_items);
        const int64_t blocks = (int64_t)t.item[t.n] * L.H;
        if (blocks == 0) continue;
        TS_TYPED((append_packed_kernel<T, HD><<<(unsigned)blocks, 256, 0, st>>>(
            L, t, d_len, static_cast<const T *>(k), k_stride, static_cast<const T *>(v), v_stride, rope, rope_pairs, n_pos)))
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_read_packed(const KvLayerView &L, const int32_t *pos0, const int32_t *off, int32_t dtype, void *k,
                              int64_t k_stride, void *v, int64_t v_stride, hipStream_t st) {
    PackTable t;
    for (int s = 0; s < L.S; s += t.n) {
        int at = s;
        pack_fill(t, off, pos0, L.S, s, [&](int n) { return read_items(pos0 ? pos0[at++] : 0, n); });
        const int64_t blocks = (int64_t)t.item[t.n] * L.H;
        if (blocks == 0) continue;
        TS_TYPED((read_packed_kernel<T, HD>
                  <<<(unsigned)blocks, 256, 0, st>>>(L, t, static_cast<T *>(k), k_stride, static_cast<T *>(v), v_stride)))
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_len_add(int32_t *d_len, int n_seq, const int32_t *off, hipStream_t st) {
    PackTable t;
    for (int s = 0; s < n_seq; s += t.n) {
        pack_fill(t, off, nullptr, n_seq, s, [](int) { return 0; });
        len_add_kernel<<<1, kPackSeqs, 0, st>>>(d_len, t);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ts
