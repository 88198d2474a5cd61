// ts_evict.hip -- eviction from the INT4 cache, for gfx950: which slots stay, by the attention they have
// received, and their rows moved together.
#include "ts_evict.h"

namespace ts {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- the choice ----------------------------------------------------------------------------------
//
// A row (one layer, sequence and kv head) keeps its first n_sink slots, its last n_recent, and of those
// between the `need` largest weights, equal ones from the lowest slot on.  Weights are compared as
// unsigned keys in their order (-0 as 0, NaN above all).

__device__ inline uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (u == 0x80000000u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Workgroup sums of one number per wave: the sum over the waves before this one, and over all.
template <int NW>
__device__ inline int wave_base(int mine, int *s, int wave, int lane, int &all) {
    __syncthreads();
    if (lane == 0) s[wave] = mine;
    __syncthreads();
    int base = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const int v = s[i];
        base += i < wave ? v : 0;
        all += v;
    }
    return base;
}

// One workgroup a row.  The keys stay in registers (of a row longer than NT * kSelPer they are read again
// for every pass).  The `need`-th largest key is found in passes over ever smaller ranges of keys: a
// histogram of kBins bins between the smallest and the largest, the bin that holds it, and so on into that bin,
// until the bin is taken whole or holds one key only.  Keys are logarithmic in the weight, so a row's spread over
// the bins also when a few slots hold most of the weight, and two passes nearly always do.
constexpr int kSelPer = 16, kBins = 2048;

template <int NT>
__global__ __launch_bounds__(NT) void select_kernel(const float *w, const int32_t *len, int n_seq, int H, int max_seq, int keep,
                                                    int n_sink, int n_recent, int32_t *slots) {
    constexpr int NW = NT / 64, E = kSelPer, TILE = NT * E, BPT = kBins / NT;
    __shared__ int hist[kBins], s_wave[NW], found[3];
    __shared__ uint32_t s_min[NW], s_max[NW];
    const size_t row = blockIdx.x;
    const int s = (int)(row / H % n_seq), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(len[s], max_seq);
    w += row * max_seq;
    slots += row * keep;
    if (n <= keep) {
        for (int j = tid; j < keep; j += NT) slots[j] = j < n ? j : -1;
        return;
    }
    const int lo = n_sink, hi = n - n_recent, tiles = (n + TILE - 1) / TILE;
    int need = keep - n_sink - n_recent;
    // element e of a tile: wave w holds slots 64 E w .. of it, in order
    const int p_lane = wave * 64 * E + lane;
    uint32_t k[E];
    auto load = [&](int t) __attribute__((always_inline)) {
        float x[E];
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = w[min(t * TILE + p_lane + 64 * e, n - 1)];
#pragma unroll
        for (int e = 0; e < E; e++) k[e] = order_key(x[e]);
    };
    auto mid = [&](int t, int e) __attribute__((always_inline)) {
        return (unsigned)(t * TILE + p_lane + 64 * e - lo) < (unsigned)(hi - lo);
    };
    if (tiles == 1) load(0);
    uint64_t sure = 0;      // keys from here on stay
    uint32_t tie = 0;       // and the first `need` of this one
    if (need > 0) {
        uint32_t base = 0xFFFFFFFFu, top = 0;
        for (int t = 0; t < tiles; t++) {
            if (tiles > 1) load(t);
#pragma unroll
            for (int e = 0; e < E; e++)
                if (mid(t, e)) {
                    base = min(base, k[e]);
                    top = max(top, k[e]);
                }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            base = min(base, (uint32_t)__shfl_xor((int)base, o, 64));
            top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        }
        if (lane == 0) {
            s_min[wave] = base;
            s_max[wave] = top;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) {
            base = min(base, s_min[i]);
            top = max(top, s_max[i]);
        }
        while (true) {
            if (base == top) {
                sure = (uint64_t)base + 1;
                tie = base;
                break;
            }
            const int shift = max(0, 32 - __clz(top - base) - 11);
#pragma unroll
            for (int i = 0; i < BPT; i++) hist[tid + NT * i] = 0;
            __syncthreads();
            for (int t = 0; t < tiles; t++) {
                if (tiles > 1) load(t);
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (mid(t, e) && k[e] >= base && k[e] <= top) atomicAdd(&hist[(k[e] - base) >> shift], 1);
            }
            __syncthreads();
            // thread t holds bins BPT t .. from the top one down
            int c[BPT], sum = 0;
#pragma unroll
            for (int i = 0; i < BPT; i++) {
                c[i] = hist[kBins - 1 - (BPT * tid + i)];
                sum += c[i];
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(upto, o, 64);
                upto += lane >= o ? v : 0;
            }
            int all;
            int above = wave_base<NW>(__shfl(upto, 63, 64), s_wave, wave, lane, all) + upto - sum;
            if (above < need && need <= above + sum) {
#pragma unroll
                for (int i = 0; i < BPT; i++) {
                    if (above < need && need <= above + c[i]) {
                        found[0] = kBins - 1 - (BPT * tid + i);
                        found[1] = above;
                        found[2] = c[i];
                    }
                    above += c[i];
                }
            }
            __syncthreads();
            const uint32_t from = base + ((uint32_t)found[0] << shift);
            need -= found[1];
            if (found[2] == need) {  // the whole bin
                sure = from;
                need = 0;
                break;
            }
            top = from + min(top - from, (1u << shift) - 1);  // (from + 2^shift may pass 2^32)
            base = from;
        }
    }
    const uint64_t below = (1ull << lane) - 1;
    int out = 0, ties = 0;
    for (int t = 0; t < tiles; t++) {
        if (tiles > 1) load(t);
        uint32_t take = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int p = t * TILE + p_lane + 64 * e;
            const bool m = mid(t, e);
            take |= (uint32_t)(m ? keep > n_sink + n_recent && k[e] >= sure : p < n) << e;
        }
        if (need > 0) {  // (uniform)
            int cnt = 0, all;
#pragma unroll
            for (int e = 0; e < E; e++) cnt += __popcll(__ballot(mid(t, e) && k[e] == tie));
            int rank = ties + wave_base<NW>(cnt, s_wave, wave, lane, all);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool eq = mid(t, e) && k[e] == tie;
                const uint64_t b = __ballot(eq);
                take |= (uint32_t)(eq && rank + __popcll(b & below) < need) << e;
                rank += __popcll(b);
            }
            ties += all;
        }
        int cnt = 0, all;
#pragma unroll
        for (int e = 0; e < E; e++) cnt += __popcll(__ballot(take >> e & 1));
        int at = out + wave_base<NW>(cnt, s_wave, wave, lane, all);
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint64_t b = __ballot(take >> e & 1);
            const int j = at + __popcll(b & below);
            if ((take >> e & 1) && j < keep) slots[j] = t * TILE + p_lane + 64 * e;
            at += __popcll(b);
        }
        out += all;
    }
}

// ---- the rows ------------------------------------------------------------------------------------
//
// Slots are ascending, so a row never moves up: the source of slot j is j or a later one.  One wave
// takes one slice of the rows of one (layer, sequence, kv head) and walks the slots in windows:
// it reads a window's sources before it writes the window, and no later window reads a slot that an
// earlier one has written, so the move needs no second copy, also in place.  Slices: the K words of
// each lane group g, 16-byte chunks of V's lane groups, the scales with the weights; they share no
// memory.  In place a slice is one wave's from its first slot to its last; into another cache the slots
// are divided among waves too.

template <int HD>
constexpr int kKeepSlices = 4 + HD / 64 + 1;
constexpr int kKeepPart = 128;  // slots of a wave that does not move in place

// Windows of STEP slots from j0 to j1, D of them in registers: window i + D - 1 goes out before window i is
// written, its slots' sources one window earlier.
template <int STEP, int D, class Reg, class Source, class Load, class Store>
__device__ __forceinline__ void walk(int j0, int j1, Source source, Load load, Store store) {
    if (j0 >= j1) return;
    Reg r[D];
    int next = source(j0);
#pragma unroll
    for (int d = 0; d < D - 1; d++) {
        const int now = next;
        next = source(j0 + STEP * (d + 1));
        if (j0 + STEP * d < j1) load(r[d], now);
    }
    int j = j0;
    while (true) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int now = next;
            next = source(j + STEP * D);
            if (j + STEP * (D - 1) < j1) load(r[(d + D - 1) % D], now);
            store(r[d], j);
            j += STEP;
            if (j >= j1) return;
        }
    }
}

template <int HD, bool IN_PLACE>
__global__ __launch_bounds__(64) void keep_kernel(KeepCall a, int n_part) {
    constexpr int NS = kKeepSlices<HD>;
    const unsigned slice = blockIdx.x % NS, part = IN_PLACE ? 0 : blockIdx.x / NS % n_part;
    const unsigned row = blockIdx.x / NS / (IN_PLACE ? 1 : n_part);
    const int lane = threadIdx.x, H = a.src.H;
    const int h = row % H, i = row / H % a.n_seq, layer = row / H / a.n_seq;
    const int len = min(a.src_len[a.src_seq + i], a.src_max), n = min(len, a.keep);
    const int j0 = IN_PLACE ? 0 : part * kKeepPart, j1 = IN_PLACE ? n : min(n, j0 + kKeepPart);
    const size_t srow = (size_t)(a.src_seq + i) * H + h, drow = (size_t)(a.dst_seq + i) * H + h;
    const int sP = a.src.P, dP = a.dst.P;
    const int32_t *slots = a.slots + (size_t)row * a.slot_row;
    const size_t so = a.src_layer * layer, dof = a.dst_layer * layer;
    // (a slot outside the source reads one inside it)
    auto source = [&](int j) __attribute__((always_inline)) { return j < n ? min(max(slots[j], 0), len - 1) : 0; };
    if (slice < 4) {
        constexpr int W = HD / 32, V = W < 4 ? W : 4, NV = W / V;  // words of a slot in lane group g, in vectors
        typedef uint32_t vec __attribute__((ext_vector_type(V)));
        struct Reg { vec x[NV]; };
        const int g = slice;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(a.src.kp + so + srow * sP * (HD / 2));
        uint32_t *dst = reinterpret_cast<uint32_t *>(a.dst.kp + dof + drow * dP * (HD / 2));
        walk<64, 4, Reg>(j0, j1, [&](int j) { return source(j + lane); },
            [&](Reg &r, int p) {
#pragma unroll
                for (int c = 0; c < NV; c++) r.x[c] = *reinterpret_cast<const vec *>(src + k_word_idx<HD>(p, 16 * c + 2 * g));
            },
            [&](const Reg &r, int j) {
                if (j + lane < n) {
#pragma unroll
                    for (int c = 0; c < NV; c++) *reinterpret_cast<vec *>(dst + k_word_idx<HD>(j + lane, 16 * c + 2 * g)) = r.x[c];
                }
            });
    } else if (slice < 4 + HD / 64) {
        struct Reg { u32x4 x[8]; int p; };
        const int td4 = slice - 4, g = lane >> 4, dl = lane & 15;
        const u32x4 *src = reinterpret_cast<const u32x4 *>(a.src.vp + so + srow * (sP / 32) * (HD * 16));
        u32x4 *dst = reinterpret_cast<u32x4 *>(a.dst.vp + dof + drow * (dP / 32) * (HD * 16));
        // slot of nibble e of this lane's words, in a block of 32
        auto slot = [&](int e) __attribute__((always_inline)) { return (e < 4 ? 0 : 16) + 4 * g + (e & 3); };
        walk<32, 3, Reg>(j0, j1, [&](int j) { return source(j + (lane & 31)); },
            [&](Reg &r, int mine) {
                r.p = mine;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int p = __shfl(mine, slot(e), 64);
                    r.x[e] = src[(size_t)(p >> 5) * HD + td4 * 64 + 16 * ((p & 15) >> 2) + dl];
                }
            },
            [&](const Reg &r, int j) {
                u32x4 x = {0, 0, 0, 0};
                uint32_t left = 0;  // nibbles of slots from n on stay
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int p = __shfl(r.p, slot(e), 64), sh = 4 * ((p & 3) + ((p & 16) >> 2));
                    const bool in = j + slot(e) < n;
                    left |= in ? 0 : 15u << (4 * e);
#pragma unroll
                    for (int c = 0; c < 4; c++) x[c] |= (r.x[e][c] >> sh & 15) << (4 * e);
                }
                u32x4 *to = dst + (size_t)(j >> 5) * HD + td4 * 64 + lane;
                if (left) {
                    const u32x4 old = *to;
#pragma unroll
                    for (int c = 0; c < 4; c++) x[c] = (x[c] & ~left) | (old[c] & left);
                }
                *to = x;
            });
    } else {
        struct Reg { float k, v, w; };
        const float *ks = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(a.src.ks) + so) + srow * sP;
        const float *vs = reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(a.src.vs) + so) + srow * sP;
        float *kd = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(a.dst.ks) + dof) + drow * dP;
        float *vd = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(a.dst.vs) + dof) + drow * dP;
        const float *ws = a.src_w ? a.src_w + ((size_t)layer * a.src.S * H + srow) * a.src_max : nullptr;
        float *wd = a.dst_w ? a.dst_w + ((size_t)layer * a.dst.S * H + drow) * a.dst_max : nullptr;
        walk<64, 4, Reg>(j0, j1, [&](int j) { return source(j + lane); },
            [&](Reg &r, int p) {
                r.k = ks[p];
                r.v = vs[p];
                r.w = wd ? ws[p] : 0.0f;
            },
            [&](const Reg &r, int j) {
                if (j + lane < n) {
                    kd[j + lane] = r.k;
                    vd[j + lane] = r.v;
                    if (wd) wd[j + lane] = r.w;
                }
            });
        // slots behind the kept ones have received nothing
        const int end = IN_PLACE ? len : a.dst_max;
        if (wd)
            for (int j = n + 64 * part + lane; j < end; j += 64 * (IN_PLACE ? 1 : n_part)) wd[j] = 0.0f;
    }
}

__global__ void keep_len_kernel(KeepCall a) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.n_seq) return;
    const int len = min(a.src_len[a.src_seq + i], a.src_max), n = min(len, a.keep), rot = a.src_rot[a.src_seq + i];
    a.dst_len[a.dst_seq + i] = n;
    a.dst_rot[a.dst_seq + i] = rot + len - n;
    a.dst_sink[a.dst_seq + i] = 0;
}

}  // namespace

hipError_t launch_select(const float *w, const int32_t *d_len, int max_len, int n_layers, int n_seq, int H, int max_seq,
                         int keep, int n_sink, int n_recent, int32_t *d_slots, hipStream_t st) {
    const unsigned rows = (unsigned)(n_layers * n_seq * H);
    // A workgroup whose registers hold the longest row, and no larger: several of the smaller one share a CU.
    if (max_len <= 256 * kSelPer)
        select_kernel<256><<<rows, 256, 0, st>>>(w, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, d_slots);
    else
        select_kernel<1024><<<rows, 1024, 0, st>>>(w, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, d_slots);
    return hipGetLastError();
}

hipError_t launch_keep(const KeepCall &c, hipStream_t st) {
    const unsigned rows = (unsigned)(c.n_layers * c.n_seq * c.src.H);
    const int n_part = (c.keep + kKeepPart - 1) / kKeepPart;
#define TS_KEEP(HDV)                                                                                          \
    {                                                                                                         \
        if (c.in_place) keep_kernel<HDV, true><<<rows * kKeepSlices<HDV>, 64, 0, st>>>(c, 1);                   \
        else keep_kernel<HDV, false><<<rows * kKeepSlices<HDV> * n_part, 64, 0, st>>>(c, n_part);               \
    }
    if (c.src.hd == 256) TS_KEEP(256)
    else if (c.src.hd == 128) TS_KEEP(128)
    else TS_KEEP(64)
#undef TS_KEEP
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    keep_len_kernel<<<(c.n_seq + 63) / 64, 64, 0, st>>>(c);
    return hipGetLastError();
}

}  // namespace ts
