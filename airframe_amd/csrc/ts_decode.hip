// ts_decode.hip -- split-K GQA decode attention over the INT4 cache for gfx950.
//
// Semantics: the CPU reference attention (src/ops/reference/attention.rs:236-313): per query
// head, scores = q.k over all cached positions, times 1/sqrt(hd), softmax, times V, with q
// rotated at its absolute position and k/v the dequantized INT4 cache
// ((code - 8) * scale, test_int4_parity.rs:78-87).  The reference GPU kernel
// (sh_layer_v1_int4.wgsl:1042-1143) runs one thread per output element, each re-reading the
// whole K stream; here the work is organised around HBM instead:
//
// * grid = (split, kv head, sequence); a split is `chunk` positions (multiple of 64) of one
//   (sequence, kv head) stream, so every workgroup reads contiguous runs of K rows, V blocks
//   and scales exactly once for all G = n_head/n_kv query heads that share them.  The chunk
//   is planned from the total context of the batch, so ragged batches get more splits for
//   their long sequences and the count of busy workgroups stays at the planned one.
// * each wave takes 64-position windows round robin; in the integer kernel every 16-byte load
//   instruction reads one contiguous kilobyte (the cache's chunk order puts each lane's K row
//   segment and V words there), non-temporally, and each workgroup starts its windows at its
//   own offset, so the concurrent streams spread over the HBM channels.
// * QK^T and PV run on the matrix cores (v_mfma_f32_16x16x32_f16).  INT4 codes convert to
//   exact f16 integers with two bit tricks (0x6400|nibble is 1024+nibble; the second nibble of
//   a byte is taken as 1024+16*nibble and fixed with one packed f16 FMA), so K and V enter the
//   MFMA exactly.  The per-position scales are applied in f32 outside the MFMA: s_k on the
//   scores, s_v folded into the probabilities.
// * q is split hi + lo in f16 (q = hi + lo to ~22 bits).  With G = n_head/n_kv <= 8 query
//   heads per kv head, 2G of the 16 MFMA columns carry the hi parts of the G heads and their
//   lo parts, so one MFMA gives both halves of every score (summed across lanes afterwards)
//   and scores carry f32-level accuracy; the probabilities enter PV split the same way.
// * online softmax in the exp2 domain with one cross-lane max per 64 positions and lazy
//   rescaling; s_v is folded into the probabilities under a per-window exponent bound so they
//   never leave f16 range.  A workgroup's waves merge through LDS; splits merge in a second
//   kernel (log-sum-exp combine) unless a sequence fits one split.
#include <stdlib.h>

#include "ts_decode_int.h"

namespace ts {
namespace {

// PAD: the caller's head dim hdr is below the stored HD (rows of q, new K/V and the output are
// hdr floats; the stored dims past them hold zeros).
// NW waves per workgroup: 4 (two workgroups per CU up to 128 dims), or 8 / 16 for a plan that
// gives every (sequence, kv head) stream one workgroup (a CU) of its own and no split: the
// small-batch case, where the combine launch would be most of the step.
template <int HD, bool SOFTCAP, bool NORM, bool PAD, int NW>
__global__ __launch_bounds__(64 * NW, NW > 4 ? 1 : (HD > 128 ? 1 : 2)) void decode_split_kernel(DecodeArgs a) {
#define TS_SPLIT_X blockIdx.x
#define TS_SPLIT_Y blockIdx.y
#define TS_SPLIT_Z blockIdx.z
#define TS_SPLIT_KEEP false
#define TS_SPLIT_SCORES false
#define TS_SPLIT_LDS                                   \
    __shared__ __align__(16) DecodeSplitSmem<HD, NW> sm; \
    __shared__ __align__(16) float kd[HD], vd[HD];       \
    __shared__ float xnew[8];
#include "ts_decode_split_body.h"
#undef TS_SPLIT_X
#undef TS_SPLIT_Y
#undef TS_SPLIT_Z
#undef TS_SPLIT_LDS
#undef TS_SPLIT_KEEP
#undef TS_SPLIT_SCORES
}

// Log-sum-exp merge of the splits of one (sequence, head).  256 threads: HD/4 threads (one
// float4 of dims each) per split row, 1024/HD row groups striding over the splits, then an
// LDS reduction over the groups, so the dependent-load chain is ns/groups long, not ns.
template <int HD>
__global__ __launch_bounds__(256) void decode_combine_kernel(DecodeArgs a) {
    const int head = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int n_ctx = (a.hlen >= 0 ? a.hlen : a.len[s]) + 1;
    const int ns = min((n_ctx + a.chunk - 1) / a.chunk, a.n_split);
    if (ns > 1) combine_rows<HD>(a, head, s, ns, tid);
    arrive_and_advance(a);
}



}  // namespace

namespace {
constexpr int kMinChunk = 256;  // splits shorter than this leave waves without a window
constexpr int kIntChunk = 1024;  // the shortest evenly spread splits that take the integer kernel

// Splits of `chunk` positions of all sequences; *idle: some sequence has fewer than the longest, whose
// grid then holds workgroups without work.
int64_t count_splits(const int32_t *n_ctx, int n_seq, int max_ctx, int chunk, bool *idle) {
    *idle = false;
    if (chunk >= max_ctx) return n_seq;
    const float inv = 1.0f / chunk;
    const int most = (max_ctx + chunk - 1) / chunk;
    int n = 0, fewer = 0;  // (32 bits and no branch: the loop runs on vectors)
    for (int s = 0; s < n_seq; s++) {
        const int c = (int)((n_ctx[s] - 0.5f) * inv) + 1;
        n += c;
        fewer |= c ^ most;
    }
    *idle = fewer != 0;
    return n;
}

// The chunk that spreads a batch's context evenly: the smallest multiple of 64 for which the busy
// workgroups of the whole batch, n_kv * sum_s ceil(n_ctx[s] / chunk), fit in `target`; with
// more streams than the target, the batch's work over the target.
int even_chunk(const int32_t *n_ctx, int n_seq, int n_kv, int target, int64_t total, int max_ctx) {
    bool idle;
    auto busy = [&](int chunk) { return count_splits(n_ctx, n_seq, max_ctx, chunk, &idle) * n_kv; };
    const int hi_c = std::max(kMinChunk, (max_ctx + 63) / 64 * 64);
    int lo_c = (int)std::min<int64_t>(hi_c, std::max<int64_t>(kMinChunk, (total * n_kv + target - 1) / target));
    lo_c = (lo_c + 63) / 64 * 64;
    int lo = lo_c / 64, hi = hi_c / 64;  // busy is non-increasing
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (busy(64 * mid) <= target) hi = mid; else lo = mid + 1;
    }
    if (busy(64 * lo) > target) return lo_c;
    return 64 * lo;
}

// What the plan weighs, in us, of either kernel: a workgroup's fixed part (lengths, q operands,
// the merge of its waves), one round of its waves (a 64-position window each, `span` positions
// together) and how many workgroups run at once.  From times of splits of 64 positions to whole
// sequences of 1 to 32 sequences of 60 to 32K positions (time against rounds of the longest
// split), all head shapes.
struct DecodeCost {
    float fixed, round;
    int span;
    float at_once;
};
// The integer kernel: one workgroup per CU; a second half of query heads makes a round half as long
// again, four halves 2.5 times (their QK^T and softmax share the wave), and all lengthen the
// fixed part (their q digits and merges).
DecodeCost int_cost(int G, int hd, int n_cu) {
    const int halves = (G + 3) / 4;
    const float heads = halves <= 1 ? 1.0f : halves == 2 ? 1.5f : 2.5f;
    const float fixed = halves <= 1 ? 5.0f : halves == 2 ? 7.5f : 13.0f;
    if (hd == 64) return {fixed, (halves <= 1 ? 1.4f : halves == 2 ? 1.8f : 3.2f), 512, (float)n_cu};
    if (hd == 256) return {fixed + 2.5f, 1.75f * heads, 256, (float)n_cu};
    return {fixed, 0.95f * heads, 256, (float)n_cu};
}
// The 16x16 kernel: two workgroups fit a CU but get in each other's way (together 1.25 times one).
DecodeCost f16_cost(int G, int hd, int n_cu) {
    const float heads = G > 4 ? 1.4f : 1.0f;
    return {4.0f, (hd == 64 ? 1.33f : hd == 128 ? 1.55f : 3.2f) * heads, 256, 1.25f * n_cu};
}
constexpr float kCombineUs = 3.5f;        // the combine launch behind a plan with splits
constexpr float kDecodeBytesUs = 6.5e6f;  // bytes a us that all CUs stream together

// Estimated time of a plan with splits of `chunk`: the longest split, or the batch's work over the
// workgroups that run at once (the last to start then ends half a split later on average), or
// the bytes.  Only 7/8 of the CUs count when the grid holds idle workgroups (splits past a
// shorter sequence's end): busy ones then wait 9-20 us for a CU that others leave, since the
// dispatcher does not place a workgroup on just any free CU of its XCD.
struct PlanTime {
    float us;
    int64_t busy, grid;  // workgroups with work, and all
    bool idle;           // some without
};
PlanTime plan_time(const DecodeCost &k, const int32_t *n_ctx, int n_seq, int streams, int64_t total, int max_ctx, int chunk,
                   int n_cu, float bytes_us) {
    PlanTime t;
    const int most = (max_ctx + chunk - 1) / chunk;
    t.busy = count_splits(n_ctx, n_seq, max_ctx, chunk, &t.idle) * streams;
    t.grid = (int64_t)most * n_seq * streams;
    const float cus = t.idle ? 0.875f : 1.0f;
    const float longest = k.fixed + k.round * ((std::min(chunk, max_ctx) + k.span - 1) / k.span);
    t.us = longest;
    if (t.busy > cus * n_cu) {
        const float work = t.busy * (k.fixed + 0.5f * k.round) + k.round * total * streams / k.span;
        t.us = std::max(t.us, work / (cus * k.at_once) + 0.5f * longest);
    }
    t.us = std::max(t.us, bytes_us + k.fixed) + (most > 1 ? kCombineUs : 0.0f);
    return t;
}

// Part of the even plan's estimate that a plan's has to stay below to take its place, 0 if it never
// does (stored: the stored head dim; even_idle: the even plan has idle workgroups).  The estimate
// knows little of how the dispatcher packs workgroups, so each kind of change has the margin with
// which its shapes keep within the runs' noise of the even plan (3%, with a few at 5), measured over
// 6000 shapes of 1 to 256 sequences of 60 to 32000 positions, equal and ragged.  (A margin of 2%
// for all left 95 of the 1064 shapes that it changed 2 to 29% slower.)
//   No split at all: 0.40 to 1.01 of the even plan's time, with less than 4% to gain up to 1.03.
//   Never the 16x16 kernel in the place of an even plan on the integer one: a tenth more error against 64
//     bits without a split, and with splits 0.83 to 1.21 of the time.
//   Splits that leave workgroups idle in a grid of more than the CUs: integer ones on 256-dim rows
//     0.41 to 0.92, on others up to 1.24; of the 16x16 kernel up to 1.20 beyond 5/8 of the CUs busy.
//   Longer splits of the 16x16 kernel: 256-dim rows 0.55 to 0.80; 128-dim rows 0.75 to 1.06, mean 0.89;
//     none on 64-dim rows (mean 0.97, up to 1.11).
//   Integer splits in the place of the 16x16 kernel's: with one half of query heads, or 256-dim rows
//     (with more halves on shorter rows 0.96 to 1.24); of fewer integer ones: 0.78 to 1.01, with less
//     to gain up to 1.11; of none: with less than a quarter to gain up to 1.29.
float plan_margin(const PlanTime &t, bool g4, bool split, const DecodePlan &even, bool even_idle, int G, int stored, int n_cu) {
    if (even.g4 && !g4) return 0.0f;
    if (!split) return even_idle ? 0.98f : 0.96f;
    if (t.idle && t.grid > n_cu && (g4 ? stored < 256 : 8 * t.busy > 5 * n_cu)) return 0.0f;
    if (!g4) return stored < 128 ? 0.0f : stored == 128 ? 0.8f : 0.98f;
    if (!even.g4) return G <= 4 || stored == 256 ? 0.98f : 0.0f;
    if (even.n_split == 1) return t.idle ? 0.0f : 0.75f;
    return stored < 128 ? 0.8f : 0.9f;
}
}  // namespace

// The batch's context spread evenly (even_chunk) over 7/8 of the CUs for the integer kernel, or, when
// its splits would be short, over twice the CUs for the 16x16 kernel.
static DecodePlan even_plan(const int32_t *n_ctx, int n_seq, int n_kv, int G, int n_cu, int stored_hd, int64_t total,
                            int max_ctx) {
    DecodePlan p;
    p.nw = 4;
    p.g4 = false;
    if (G <= decode_int_gmax(stored_hd)) {
        p.chunk = even_chunk(n_ctx, n_seq, n_kv, n_cu - n_cu / 8, total, max_ctx);
        p.g4 = p.chunk >= kIntChunk;
    }
    if (!p.g4) p.chunk = even_chunk(n_ctx, n_seq, n_kv * ((G + 7) / 8), 2 * n_cu, total, max_ctx);
    p.n_split = p.even_split = (max_ctx + p.chunk - 1) / p.chunk;
    return p;
}

static void context_of(const int32_t *n_ctx, int n_seq, int64_t &total, int &max_ctx) {
    total = 0;
    max_ctx = 1;
    for (int s = 0; s < n_seq; s++) {
        max_ctx = std::max(max_ctx, (int)n_ctx[s]);
        total += n_ctx[s];
    }
}

DecodePlan decode_plan_even(const int32_t *n_ctx, int n_seq, int n_kv, int G, int n_cu, int stored_hd) {
    int64_t total;
    int max_ctx;
    context_of(n_ctx, n_seq, total, max_ctx);
    return even_plan(n_ctx, n_seq, n_kv, G, n_cu, stored_hd, total, max_ctx);
}

// Split plan: the kernel and the split length whose estimate is the lowest, among the batch's
// context spread evenly (decode_plan_even) and equal shares of the longest sequence, fewest first;
// a later one in that order has to gain 2%, and all of them the margin that their kind has over
// the even plan (plan_margin).  (The even plan alone gave a ragged batch of about as
// many streams as CUs a few second splits, which waited for the first ones, with a combine behind
// them and idle workgroups between.  32 sequences of 700-1531 positions, 8 kv heads: 27.3 us with
// two splits for some, 17.8 with none; 2000-6000: 36.4, 30.1; 64-dim rows, 1000-3000: 22.1, 13.2.
// And the integer kernel took only splits of 1024 and more: 8 sequences of 1000-4000 positions
// with 256-dim rows 36.2 us on the 16x16 kernel, 19.3 in integer splits of 832; one sequence of
// 20000 with 24 query heads 17.2 us a layer, 12.4.)
DecodePlan decode_plan(const int32_t *n_ctx, int n_seq, int n_kv, int G, int n_cu, int stored_hd, bool fused) {
    int max_ctx;
    int64_t total;
    context_of(n_ctx, n_seq, total, max_ctx);
    DecodePlan p;
    p.nw = 4;
    const int groups = (G + 7) / 8;  // head groups of the 16x16 kernel
    // Few streams, short context: one wide workgroup of the 16x16 kernel per stream instead of a
    // split, when its waves cover the longest sequence's windows (the positions before the new
    // token with the fused append, which scores that one from registers) in one round.  No
    // combine launch (the split kernel then also advances the lengths), the merge stays in LDS.
    // The fewest waves that cover it: 8 waves measured 9.1 us per step on config 1's shape (512
    // positions + the new token), 16 waves 10.1, four-wave splits and a combine 10.5.  More than
    // one window per wave does not pay: 8.5 windows per wave took 26.6 us per layer on config 2's
    // shape against 10.0 with splits and a combine.
    // (Not in the place of the integer kernel without a split, which serves about as many streams as
    // CUs: 256 streams of 1000 64-dim positions 9.8 us a layer, 12.6 with 16 waves.  Shorter contexts
    // need no even plan to know.)
    auto integer_even = [&] {
        return (max_ctx + 63) / 64 * 64 >= kIntChunk && even_plan(n_ctx, n_seq, n_kv, G, n_cu, stored_hd, total, max_ctx).g4;
    };
    const int n_win = (max_ctx - (fused ? 1 : 0) + 63) / 64;
    const int wmax = stored_hd <= 64 ? 16 : stored_hd <= 128 ? 8 : 4;
    if (n_win > 4 && n_win <= wmax && (int64_t)n_seq * n_kv * groups <= n_cu && !integer_even()) {
        p.g4 = false;
        p.nw = n_win <= 8 ? 8 : 16;
        p.chunk = (max_ctx + 63) / 64 * 64;
        p.n_split = p.even_split = 1;
        return p;
    }
    const float bytes_us = (float)total * n_kv * (stored_hd + 8) / kDecodeBytesUs;
    const bool integer = G <= decode_int_gmax(stored_hd);
    const DecodeCost ki = int_cost(G, stored_hd, n_cu), kf = f16_cost(G, stored_hd, n_cu);
    const DecodePlan even = even_plan(n_ctx, n_seq, n_kv, G, n_cu, stored_hd, total, max_ctx);
    auto time = [&](int chunk, bool g4) {
        return plan_time(g4 ? ki : kf, n_ctx, n_seq, n_kv * (g4 ? 1 : groups), total, max_ctx, chunk, n_cu, bytes_us);
    };
    const PlanTime even_t = time(even.chunk, even.g4);
    p = even;
    float best = even_t.us;
    auto weigh = [&](int chunk, bool g4) {
        const PlanTime t = time(chunk, g4);
        if (t.us < 0.98f * best &&
            t.us < plan_margin(t, g4, chunk < max_ctx, even, even_t.idle, G, stored_hd, n_cu) * even_t.us) {
            best = t.us;
            p.g4 = g4;
            p.chunk = chunk;
        }
    };
    // (no plan is estimated below the bytes and either kernel's fixed part)
    if (0.98f * best <= bytes_us + std::min(ki.fixed, kf.fixed)) return p;
    const int most = std::min((max_ctx + kMinChunk - 1) / kMinChunk, decode_cap(n_kv, max_ctx, n_cu));
    for (int k = 1; k <= most; k = k == most ? k + 1 : std::min(most, k + (k < 8 ? 1 : k / 4))) {
        // (a few positions to spare, so that the plan of a length that is a multiple of k windows
        // outlives the next tokens, as a captured one has to)
        const int chunk = ((max_ctx + k - 1) / k + (k > 1 ? 4 : 0) + 63) / 64 * 64;
        if (integer) weigh(chunk, true);
        weigh(chunk, false);
    }
    p.n_split = (max_ctx + p.chunk - 1) / p.chunk;
    return p;
}

int decode_cap(int n_kv, int max_seq, int n_cu) {
    // One sequence alone can take at most target / n_kv splits (plus one for rounding); the
    // 16x16 kernel's target, 2 n_cu, is the larger.
    return std::min((max_seq + 63) / 64, 2 * n_cu / n_kv + 2);
}

namespace {
template <int HD, bool SC, bool NM, bool PAD>
void launch_16x16_pad(const DecodeArgs &a, dim3 grid, int nw, hipStream_t st) {
    if (HD <= 128 && nw == 8)
        decode_split_kernel<HD, SC, NM, PAD, HD <= 128 ? 8 : 4><<<grid, 64 * 8, 0, st>>>(a);
    else if (HD <= 64 && nw == 16)
        decode_split_kernel<HD, SC, NM, PAD, HD <= 64 ? 16 : 4><<<grid, 64 * 16, 0, st>>>(a);
    else
        decode_split_kernel<HD, SC, NM, PAD, 4><<<grid, 64 * 4, 0, st>>>(a);
}

template <int HD, bool SC, bool NM>
void launch_16x16(const DecodeArgs &a, dim3 grid, int nw, bool pad, hipStream_t st) {
    if (pad) launch_16x16_pad<HD, SC, NM, true>(a, grid, nw, st);
    else launch_16x16_pad<HD, SC, NM, false>(a, grid, nw, st);
}

}  // namespace

hipError_t launch_decode(const KvLayerView &L, int32_t *d_len, const int32_t *h_len, const float *q, int n_head,
                         const float *rope, int rope_pairs, float softcap, float *out,
                         float *ws, const DecodePlan &plan, const float *k_new,
                         const float *v_new, int32_t *adv, hipStream_t st) {
    DecodeArgs a;
    a.L = L;
    a.len = d_len;
    a.hlen = h_len && L.S == 1 ? h_len[0] : -1;
    a.q = q;
    a.rope = rope;
    a.rope_pairs = rope_pairs;
    a.n_head = n_head;
    a.Gt = n_head / L.H;
    a.NG = plan.g4 ? 1 : (a.Gt + 7) / 8;
    a.G = plan.g4 ? a.Gt : std::min(a.Gt, 8);
    a.chunk = plan.chunk;
    a.n_split = plan.n_split;
    a.inv_sqrt_hd = 1.0f / sqrtf((float)L.hdr);
    a.softcap = softcap;
    a.out = out;
    a.ws = ws;
    a.k_new = k_new;
    a.v_new = v_new;
    a.inv_softcap = 0.0f;
    a.scores = a.w = nullptr;
    a.max_seq = 0;
    a.fresh = false;
    // with a split the combine kernel advances the lengths (the last of its workgroups to
    // arrive); without one a length update follows the decode launch
    // (the 16x16 kernel does it itself when there is no split)
    const bool adv_in_kernel = plan.n_split > 1 || !plan.g4;
    a.adv_len = adv && adv_in_kernel ? d_len : nullptr;
    a.adv_ctr = adv && adv_in_kernel ? adv : nullptr;
    dim3 grid(plan.n_split, L.H * a.NG, L.S);
    // The integer kernel (plan.g4) does less VALU work per window than the 16x16 one but has the
    // longer per-window dependency chain.
    const bool cap = softcap > 0.0f, norm = L.qn != nullptr || L.kn != nullptr;
    const bool pad = L.hdr != L.hd;
#define TS_SPLIT(HDV, SC, NM)                                                                  \
    (plan.g4 ? (launch_integer<HDV, SC, NM>(a, plan.n_split, pad, a.Gt, st), 0) \
             : (launch_16x16<HDV, SC, NM>(a, grid, plan.nw, pad, st), 0))
#define TS_SPLIT_HD(HDV)                                                                      \
    (cap ? (norm ? TS_SPLIT(HDV, true, true) : TS_SPLIT(HDV, true, false))                    \
         : (norm ? TS_SPLIT(HDV, false, true) : TS_SPLIT(HDV, false, false)))
    if (L.hd == 256) {
        TS_SPLIT_HD(256);
        if (plan.n_split > 1) decode_combine_kernel<256><<<dim3(n_head, L.S), 256, 0, st>>>(a);
    } else if (L.hd == 128) {
        TS_SPLIT_HD(128);
        if (plan.n_split > 1) decode_combine_kernel<128><<<dim3(n_head, L.S), 256, 0, st>>>(a);
    } else if (L.hd == 64) {
        TS_SPLIT_HD(64);
        if (plan.n_split > 1) decode_combine_kernel<64><<<dim3(n_head, L.S), 256, 0, st>>>(a);
    } else {
        return hipErrorInvalidValue;
    }
#undef TS_SPLIT_HD
#undef TS_SPLIT
    if (adv && !adv_in_kernel) {
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        return launch_len_update(d_len, L.S, -1, 1, 0, st);
    }
    return hipGetLastError();
}

}  // namespace ts
