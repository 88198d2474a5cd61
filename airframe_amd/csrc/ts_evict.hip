// ts_evict.hip -- eviction from the INT4 cache, for gfx950: which slots stay, by the attention they have
// received, and their rows moved together.
#include "ts_evict.h"

#include <algorithm>

namespace ts {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- the choice ----------------------------------------------------------------------------------
//
// A row (one layer, sequence and kv head) keeps its first n_sink slots, its last n_recent, and of those
// between the `need` largest weights, equal ones from the lowest slot on.  Weights are compared as
// unsigned keys in their order (-0 as 0, NaN above all).

__device__ inline uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);  // (-0 + 0 is 0)
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return w != w ? 0xFFFFFFFFu : k;
}

// op over the 64 lanes of a wave, every lane getting the result: DPP within each 16-lane row, then two permlane swaps.
template <int CTRL>
__device__ inline uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
template <class Op>
__device__ inline uint32_t wave_all(uint32_t v, Op op) {
    v = op(v, dpp_u<0xB1>(v));   // quad_perm(1,0,3,2)
    v = op(v, dpp_u<0x4E>(v));   // quad_perm(2,3,0,1)
    v = op(v, dpp_u<0x141>(v));  // row_half_mirror
    v = op(v, dpp_u<0x140>(v));  // row_mirror
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op(b[0], b[1]);
}

// The sum over the lanes up to this one.
__device__ inline int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8: within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// One number per wave: the sum over the waves before this one, and over all.  (A barrier between two calls.)
template <int NW>
__device__ inline int wave_base(int mine, int *s, int wave, int lane, int &all) {
    if (lane == 0) s[wave] = mine;
    __syncthreads();
    const int v = wave_scan(lane < NW ? s[lane] : 0);
    all = __builtin_amdgcn_readlane(v, NW - 1);
    return wave > 0 ? __builtin_amdgcn_readlane(v, wave - 1) : 0;
}

// One workgroup a row; the slots between the first n_sink and the last n_recent compete.  Their keys stay in
// registers (of a row longer than NT * kSelPer they are read again for every pass).  The `need`-th largest key is found in
// passes over ever smaller ranges of keys: a histogram of kBins bins between the smallest and the largest, the bin that
// holds it, and so on into that bin, until the bin is taken whole or holds one key only.  Keys are logarithmic in the
// weight, so a row's spread over the bins also when a few slots hold most of the weight, and two passes nearly
// always do.  The chosen slots go through LDS, so that a wave writes lines: written by the thread that found them, 4096
// of 4352 slots of 2304 rows took 53 us, 26 so.
//   A few rows are bound by that chain (28 of 4096 slots: 9 us), many by HBM and the rounds of the CUs: 2304 rows
// of 16000 slots 47 us, 3.1 TB/s.
constexpr int kSelPer = 16, kBins = 2048;

template <int NT>
__global__ __launch_bounds__(NT, NT == 256 ? 7 : 8) void select_kernel(const float *weights, const int32_t *len, int n_seq, int H, int max_seq,
                                                       int keep, int n_sink, int n_recent, int32_t *slots) {
    constexpr int NW = NT / 64, E = kSelPer, TILE = NT * E, BPT = kBins / NT;
    __shared__ int hist[kBins > TILE / 2 ? kBins : TILE / 2], s_wave[3][NW], found[3];  // hist: then a tile's chosen slots
    __shared__ uint32_t s_min[NW], s_max[NW];
    const size_t row = blockIdx.x;
    const int s = (int)(row / H % n_seq), tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = min(len[s], max_seq);
    slots += row * keep;
    if (n <= keep) {
        for (int j = tid; j < keep; j += NT) slots[j] = j < n ? j : -1;
        return;
    }
    const int m = n - n_sink - n_recent;  // slots that compete
    int need = keep - n_sink - n_recent;
    for (int j = tid; j < n_sink; j += NT) slots[j] = j;
    for (int j = tid; j < n_recent; j += NT) slots[keep - n_recent + j] = n - n_recent + j;
    if (need == 0) return;
    const __amdgpu_buffer_rsrc_t w =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(weights + row * max_seq + n_sink), (short)0, m * 4, 0x00020000);
    const int tiles = (m + TILE - 1) / TILE;
    // thread i of a tile holds slots E i .., in order; 0, which is no key, past the last one
    uint32_t k[E];
    auto load = [&](int t) __attribute__((always_inline)) {
        const int p = t * TILE + tid * E;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(w, 4 * p + 4 * e, 0, 0);
#pragma unroll
            for (int c = 0; c < 4; c++) k[e + c] = x[c];
        }
#pragma unroll
        for (int e = 0; e < E; e++) k[e] = p + e < m ? order_key(__uint_as_float(k[e])) : 0;
    };
    load(0);
    uint32_t base = 0xFFFFFFFFu, top = 0;
    for (int t = 0; t < tiles; t++) {
        if (t > 0) load(t);
#pragma unroll
        for (int e = 0; e < E; e++) {
            base = min(base, k[e] - 1);  // (0 becomes the largest)
            top = max(top, k[e]);
        }
    }
    base = wave_all(base, [](uint32_t a, uint32_t b) { return min(a, b); });
    top = wave_all(top, [](uint32_t a, uint32_t b) { return max(a, b); });
    if (lane == 0) {
        s_min[wave] = base;
        s_max[wave] = top;
    }
#pragma unroll
    for (int i = 0; i < BPT; i++) hist[tid + NT * i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; i++) {
        base = min(base, s_min[i]);
        top = max(top, s_max[i]);
    }
    base++;
    uint32_t tie = 0;   // the first `need` of this key stay,
    uint32_t over = 0;  // and all above this one (at least 1 below the smallest key)
    while (true) {
        if (base == top) {
            over = tie = base;
            break;
        }
        const uint32_t span = top - base;
        const int shift = max(0, 32 - __clz(span) - 11);
        for (int t = 0; t < tiles; t++) {
            if (tiles > 1) load(t);
#pragma unroll
            for (int e = 0; e < E; e++)
                if (k[e] - base <= span) atomicAdd(&hist[(k[e] - base) >> shift], 1);
        }
        __syncthreads();
        // thread t holds bins BPT t .. from the top one down
        int c[BPT], sum = 0;
#pragma unroll
        for (int i = 0; i < BPT; i++) {
            int *b = &hist[kBins - 1 - (BPT * tid + i)];
            c[i] = *b;
            *b = 0;  // (for the next pass)
            sum += c[i];
        }
        const int upto = wave_scan(sum);
        int all;
        int above = wave_base<NW>(__builtin_amdgcn_readlane(upto, 63), s_wave[0], wave, lane, all) + upto - sum;
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
        base += (uint32_t)found[0] << shift;
        need -= found[1];
        if (found[2] == need) {  // the whole bin
            over = base - 1;
            need = 0;
            break;
        }
        top = base + min(top - base, (1u << shift) - 1);  // (base + 2^shift may pass 2^32)
    }
    slots += n_sink;
    const int most = keep - n_sink - n_recent;
    int out = 0, ties = 0;
    for (int t = 0; t < tiles; t++) {
        if (tiles > 1) load(t);
        uint32_t take = 0;
#pragma unroll
        for (int e = 0; e < E; e++) take |= (uint32_t)(k[e] > over) << e;
        if (need > 0) {  // (uniform)
            uint32_t eq = 0;
#pragma unroll
            for (int e = 0; e < E; e++) eq |= (uint32_t)(k[e] == tie) << e;
            const int upto = wave_scan(__popc(eq));
            int all, rank = ties + upto - __popc(eq);
            rank += wave_base<NW>(__builtin_amdgcn_readlane(upto, 63), s_wave[1], wave, lane, all);
            for (; eq && rank < need; eq &= eq - 1, rank++) take |= eq & -eq;
            ties += all;
        }
        const int upto = wave_scan(__popc(take));
        int all, at = upto - __popc(take);
        at += wave_base<NW>(__builtin_amdgcn_readlane(upto, 63), s_wave[2], wave, lane, all);
        uint16_t *const list = reinterpret_cast<uint16_t *>(hist);
        for (; take; take &= take - 1) list[at++] = (uint16_t)(tid * E + __builtin_ctz(take));
        __syncthreads();
        const int now = min(all, most - out);
        for (int i = tid; i < now; i += NT) slots[out + i] = n_sink + t * TILE + list[i];
        out += all;
        __syncthreads();  // (the list and the waves' counts are read before the next tile's)
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
//   Elsewhere it is bound by HBM, whose lines a gather reads for the slots between too: 2048 of 2048-8192 slots of 4
// layers, 8 sequences, 8 heads of 128 dims 56 us, 143 MB of kept rows read and written, 262 MB with the slots
// between (counted, 4.7 TB/s).  In place a wave's
// instructions over its windows bound a lone layer (4096 of 4352 slots: 104 us), HBM many (36 layers of 8 sequences: 823
// us, 3.2 TB/s); with eight windows of K and five of V on their way instead of four and three 101 and 990 us.

template <int HD>
constexpr int kKeepSlices = 4 + HD / 64 + 1;
// Slots of a wave that does not move in place: one window of K, so that the launch's waves and not a wave's registers hold what
// is on its way (128 slots: 59.5 us against 56 in the case above, 6.9 and 6.5 of 4 sequences of 2 layers).
constexpr int kKeepPart = 64;

// Windows of STEP slots from j0 to j1, D of them in registers: window i + D - 1 is asked for before window i is
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

// Sequence i's length, window base (new tokens go on at the positions they would have had) and sinks.
__device__ inline void set_length(const KeepCall &a, int i, int len, int n) {
    a.dst_len[a.dst_seq + i] = n;
    a.dst_rot[a.dst_seq + i] = a.src_rot[a.src_seq + i] + len - n;
    a.dst_sink[a.dst_seq + i] = 0;
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
    const size_t so = a.src_layer * (a.first_layer + layer), dof = a.dst_layer * (a.first_layer + layer);
    // (in place the lengths change behind the launch: its other workgroups read them)
    if (!IN_PLACE && slice == 0 && part == 0 && layer == 0 && h == 0 && lane == 0) set_length(a, i, len, n);
    // (a slot outside the source reads one inside it)
    auto source = [&](int j) __attribute__((always_inline)) { return j < n ? min(max(slots[j], 0), len - 1) : 0; };
    if (slice < 4) {
        constexpr int W = HD / 32, V = W < 4 ? W : 4, NV = W / V;  // words of a slot in lane group g, in vectors
        typedef uint32_t vec __attribute__((ext_vector_type(V)));
        struct Reg { vec x[NV]; };
        const int g = slice;
        const uint32_t *src = reinterpret_cast<const uint32_t *>(a.src.kp + so + srow * sP * (HD / 2));
        uint32_t *dst = reinterpret_cast<uint32_t *>(a.dst.kp + dof + drow * dP * (HD / 2));
        walk<64, IN_PLACE ? 4 : 1, Reg>(j0, j1, [&](int j) { return source(j + lane); },
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
        walk<32, IN_PLACE ? 3 : 1, Reg>(j0, j1, [&](int j) { return source(j + (lane & 31)); },
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
        walk<64, IN_PLACE ? 4 : 1, Reg>(j0, j1, [&](int j) { return source(j + lane); },
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
        const int end = IN_PLACE && a.src_w == a.dst_w ? len : a.dst_max;
        if (wd)
            for (int j = n + 64 * part + lane; j < end; j += 64 * (IN_PLACE ? 1 : n_part)) wd[j] = 0.0f;
    }
}

__global__ void keep_len_kernel(KeepCall a) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.n_seq) return;
    const int len = min(a.src_len[a.src_seq + i], a.src_max);
    set_length(a, i, len, min(len, a.keep));
}

}  // namespace

// Layers of one launch: its work-items are a 32-bit number.
static int layers_per_launch(int64_t items, int n_layers) { return (int)std::min<int64_t>(std::max<int64_t>(1, UINT32_MAX / items), n_layers); }

hipError_t launch_select(const float *w, const int32_t *d_len, int max_len, int n_layers, int n_seq, int H, int max_seq,
                         int keep, int n_sink, int n_recent, int32_t *d_slots, hipStream_t st) {
    const int64_t rows = (int64_t)n_seq * H;
    // A workgroup whose registers hold the longest row, and no larger: several of the smaller ones share a CU.  2304 rows
    // with 256, 512 and 1024 threads: of 4096 slots 22.8, 25.2, 40.1 us, of 8192 50.4, 25.4, 40.7, of 16000 99.7, 89.6, 47.1.
    const int nt = max_len <= 256 * kSelPer ? 256 : max_len <= 512 * kSelPer ? 512 : 1024;
    const int per = layers_per_launch(rows * nt, n_layers);
    for (int i = 0; i < n_layers; i += per) {
        const unsigned wgs = (unsigned)(std::min(per, n_layers - i) * rows);
        const float *wi = w + i * rows * max_seq;
        int32_t *to = d_slots + i * rows * keep;
        if (nt == 256) select_kernel<256><<<wgs, 256, 0, st>>>(wi, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, to);
        else if (nt == 512) select_kernel<512><<<wgs, 512, 0, st>>>(wi, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, to);
        else select_kernel<1024><<<wgs, 1024, 0, st>>>(wi, d_len, n_seq, H, max_seq, keep, n_sink, n_recent, to);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int HD>
static hipError_t launch_rows(KeepCall c, hipStream_t st) {
    const int64_t rows = (int64_t)c.n_seq * c.src.H;
    const int n_part = c.in_place ? 1 : (c.keep + kKeepPart - 1) / kKeepPart, n_layers = c.n_layers;
    const int per = layers_per_launch(rows * kKeepSlices<HD> * n_part * 64, n_layers);
    for (int i = 0; i < n_layers; i += per) {
        c.n_layers = std::min(per, n_layers - i);
        const unsigned wgs = (unsigned)(c.n_layers * rows * kKeepSlices<HD> * n_part);
        if (c.in_place) keep_kernel<HD, true><<<wgs, 64, 0, st>>>(c, 1);
        else keep_kernel<HD, false><<<wgs, 64, 0, st>>>(c, n_part);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        c.first_layer += per;
        c.slots += per * rows * c.slot_row;
        if (c.dst_w) {
            c.src_w += (int64_t)per * c.src.S * c.src.H * c.src_max;
            c.dst_w += (int64_t)per * c.dst.S * c.dst.H * c.dst_max;
        }
    }
    return hipSuccess;
}

hipError_t launch_keep(const KeepCall &c, hipStream_t st) {
    const hipError_t e = c.src.hd == 256 ? launch_rows<256>(c, st) : c.src.hd == 128 ? launch_rows<128>(c, st) : launch_rows<64>(c, st);
    if (e != hipSuccess || !c.in_place) return e;
    keep_len_kernel<<<(c.n_seq + 63) / 64, 64, 0, st>>>(c);
    return hipGetLastError();
}

}  // namespace ts
