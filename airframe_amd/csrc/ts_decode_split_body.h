// ts_decode_split_body.h -- the body of decode_split_kernel (ts_decode.hip) and of decode_split
// (ts_decode_split.h): one split of one (sequence, kv head) stream in the 16x16 decode kernel.  Text and
// not a function: as an inlined function the decode kernels were scheduled otherwise, and up to 4%
// slower (16 sequences of 2801-4403 256-dim positions, 26.7 -> 27.7 us).
// In scope: HD, SOFTCAP, NORM, PAD, NW, a; TS_SPLIT_X, _Y, _Z: the split, the kv head and group of query
// heads, the sequence; TS_SPLIT_LDS: declares sm (DecodeSplitSmem), kd, vd and xnew; TS_SPLIT_KEEP: partials
// also of a sequence without a split (a flag in the arguments cost the decode kernels 2%).
    constexpr int SPAN = 64 * NW;     // positions one round of windows covers
    constexpr int WPG = HD / 32;   // K words per lane group = MFMA k-steps per 16-row tile
    constexpr int NTD = HD / 16;   // 16-dim output tiles
    constexpr int ROWB = HD / 2;   // bytes per K row
    constexpr int OST = HD + 4;  // 16-byte rows of the merge area
    const KvLayerView &L = a.L;
    const int hdr = PAD ? L.hdr : HD;
    const float *const QN = NORM ? L.qn : nullptr;  // QK norm of q (compiled out when off)
    const int split = TS_SPLIT_X, s = TS_SPLIT_Z;
    // kv head h, and head group gi of its a.Gt query heads (groups of 8)
    const int h = TS_SPLIT_Y / a.NG, gi = TS_SPLIT_Y - h * a.NG;
    const int start = split * a.chunk;
    const int tid = threadIdx.x, lane = tid & 63;
    // wave index in an SGPR: window bases are then provably wave-uniform and feed the scalar
    // offset of the buffer loads directly
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int G = min(a.G, a.Gt - 8 * gi);  // query heads of this workgroup
    const int hb = h * a.Gt + 8 * gi;       // the first of them within the sequence
    const size_t row = (size_t)s * L.H + h;
    const uint8_t *kbase = L.kp + row * L.P * ROWB;
    const uint8_t *vbase = L.vp + row * (L.P / 32) * (HD * 16);
    const float *ksb = L.ks + row * L.P;
    const float *vsb = L.vs + row * L.P;

    // The first window and the raw q go out before the sequence's length is known (a memory
    // round trip of its own): the first window is bounded by the stream's capacity, and the
    // positions of it past the split's end are masked like any tail.
    Streams str;
    str.k = make_rsrc(kbase, (uint32_t)L.P * ROWB);
    str.v = make_rsrc(vbase, (uint32_t)(L.P / 32) * (HD * 16));
    str.ksb = ksb;
    str.vsb = vsb;
    str.last = L.P - 1;
    Window<HD> w0, w1;
    int base = start + wave * 64;
    load_window<HD>(w0, str, base, n, g, lane);
    // accumulator column n: high parts of head h*G + n (n < G), low parts of head
    // h*G + n - G (G <= n < 2G), unused beyond
    const bool live = n < 2 * G, lo_col = n >= G;
    const int qhead = n < G ? n : (live ? n - G : 0);
    const float *qrow = a.q + ((size_t)s * a.n_head + hb + qhead) * hdr;
    float qraw[WPG][8];
#pragma unroll
    for (int t = 0; t < WPG; t++) q_read8(qrow, k16_word<HD>(g, t), nullptr, 1.0f, qraw[t], hdr);
    asm volatile("" ::: "memory");

    const int qpos = a.hlen >= 0 ? a.hlen : a.len[s];
    // a captured launch replayed past the cache's capacity (the host checks lengths only when a
    // call is made): no work, nothing written (the lengths still advance, as the combine
    // kernel's do)
    if (qpos >= L.P) {
        if (a.n_split == 1) arrive_and_advance(a);
        return;
    }
    const int qrot = rot_of(a.L, s, qpos);  // rotation position of the query
    const int n_ctx = qpos + 1;
    if (start >= n_ctx) return;  // (only with a split: its combine kernel advances the lengths)
    const int n_split_s = min((n_ctx + a.chunk - 1) / a.chunk, a.n_split);
    // With the fused append, this split's workgroup writes position qpos itself and adds its
    // score from registers; the window loop then stops short of it.
    const bool fused = a.k_new != nullptr && split == n_split_s - 1;
    // the last split runs to the end, also past chunk * n_split (a launch captured for shorter
    // contexts stays correct, only less balanced)
    const int end = fused ? qpos : (split == n_split_s - 1 ? n_ctx : start + a.chunk);
    const int partner4 = 4 * (n < G ? lane + G : (live ? lane - G : lane));
    const DeqConst dc;

    TS_SPLIT_LDS

    // Later windows: bounded to the split (K rows are cut into segments spread over their
    // 64-position window: bound at the window)
    str.k = make_rsrc(kbase, (uint32_t)((end + 63) & ~63) * ROWB);
    str.v = make_rsrc(vbase, (uint32_t)((end + 31) / 32) * (HD * 16));
    str.last = max(end - 1, 0);

    // q operands: wave w builds k-step t = w (rotated, scaled by log2(e)/sqrt(hd), split hi/lo)
    // for all 64 lanes; zero in the columns past G.
    // One power-of-two scale for the G heads: every wave reads the bound of all of them.
    // QK norm scale of this lane's query head (each wave computes it for itself)
    const float ns = QN ? q_norm_scale_wave<HD>(a.q + ((size_t)s * a.n_head + hb) * hdr, G, qhead, L.norm_eps, hdr)
                        : 1.0f;
    if (QN) {
#pragma unroll
        for (int t = 0; t < WPG; t++)
            if (8 * k16_word<HD>(g, t) < hdr) {
#pragma unroll
                for (int e = 0; e < 8; e++) qraw[t][e] = qk_norm_apply(qraw[t][e], ns, QN[8 * k16_word<HD>(g, t) + e]);
            }
    }
    float q_s, inv_s;
    {
        float qb = 0.0f;
#pragma unroll
        for (int t = 0; t < WPG; t++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) qb = fmaxf(qb, fabsf(qraw[t][e]) + fabsf(qraw[t][e + 1]));
        q_scale(wave_max(qb) * (a.inv_sqrt_hd * kLog2e), q_s, inv_s);
    }
#pragma unroll
    for (int t = 0; t < WPG; t++) {
        if (t % NW != wave) continue;
        half8 qh, ql;
        float2 cs[4];
        load_rot8(a.rope, a.rope_pairs, k16_word<HD>(g, t), qrot, cs);
        split_q8(qraw[t], cs, k16_word<HD>(g, t), a.rope_pairs, a.inv_sqrt_hd * kLog2e * q_s, qh, ql);
        sm.run.q.p[t][lane] = !live ? (half8)(_Float16)0.0f : (lo_col ? ql : qh);
    }
    __syncthreads();  // q operands
    // The appending wave (the last: it has the fewest windows) quantizes the new token and
    // scores it against every head before its windows; the others start at once.  kd, vd and
    // xnew are read after the barrier that opens the merge.
    if (fused && wave == NW - 1) {
        AppendIn<HD> ain;
        float2 qp[8][AppendIn<HD>::PPL];
        append_load<HD, NORM>(a, s, h, qpos, lane, ain, hdr);
        load_q_pairs<HD, 8>(a, s, hb, G, lane, qp, hdr);
        append_store<HD, NORM>(a, s, h, qpos, lane, ain, kd, vd, hdr, gi == 0);
        new_token_scores<HD, SOFTCAP, NORM, 8>(a, s, hb, G, lane, qp, ain.cs, kd, xnew, hdr);
    }

    WaveState<HD> st;
#pragma unroll
    for (int td = 0; td < NTD; td++) st.o[td] = (floatx4)0.0f;
    st.m = kMinit;
    st.l = 0.0f;
    float *stage = sm.run.stage[wave];

    // Register double buffering: window i+1 is in flight while window i is computed.  One form
    // for every window, the tail mask included (a masked and an unmasked copy cost 70 VGPRs
    // in moves at their join).
#define TS_STEP(CUR, NXT)                                                                       \
    {                                                                                          \
        load_window<HD>(NXT, str, base + SPAN, n, g, lane);                                     \
        /* keep the prefetch here: the scheduler would otherwise sink it below CUR's use */     \
        asm volatile("" ::: "memory");                                                         \
        __builtin_amdgcn_sched_barrier(0);                                                     \
        process_window<HD, SOFTCAP>(CUR, st, sm.run.q, stage, base, end, lane, g, live, lo_col, partner4, inv_s, a.softcap, dc); \
        base += SPAN;                                                                           \
        if (base >= end) break;                                                                \
    }
    while (base < end) {
        TS_STEP(w0, w1)
        TS_STEP(w1, w0)
    }
#undef TS_STEP

    // ---- merge the waves through LDS -----------------------------------------------------------
    // Each wave writes its O^T columns (16-byte stores), m and l; one barrier; then one float4
    // of dims per thread.  (Merge area shared with the q operands, a barrier before the writes,
    // scalar stores and one dim per thread: 0.1-0.3 us more per layer on configs 1 and 2.)
    const float l_run = group_sum(st.l);
    if (live) {
        if (g == 0 && !lo_col) {
            sm.merge.m[wave][n] = st.m;
            sm.merge.l[wave][n] = l_run;
        }
#pragma unroll
        for (int td = 0; td < NTD; td++)
            *reinterpret_cast<floatx4 *>(&sm.merge.o[wave][n * OST + 16 * td + 4 * g]) = st.o[td];
    }
    __syncthreads();

    constexpr int V4 = HD / 4;
    for (int idx = tid; idx < G * V4; idx += SPAN) {
        const int hh = idx / V4, d = 4 * (idx % V4);
        float M = kMinit;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, sm.merge.m[w][hh]);
        if (fused) M = fmaxf(M, xnew[hh]);
        floatx4 acc = (floatx4)0.0f;
        float lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float e = exp2f(sm.merge.m[w][hh] - M);
            const floatx4 hi = *reinterpret_cast<const floatx4 *>(&sm.merge.o[w][hh * OST + d]);
            const floatx4 lo = *reinterpret_cast<const floatx4 *>(&sm.merge.o[w][(hh + G) * OST + d]);
            acc += e * (hi + lo);
            lsum += e * sm.merge.l[w][hh];
        }
        if (fused) {
            // the new position as one more partial: m = its score, l = 1, o = its V row
            const float e = exp2f(xnew[hh] - M);
            acc += e * *reinterpret_cast<const floatx4 *>(&vd[d]);
            lsum += e;
        }
        const size_t head = (size_t)s * a.n_head + hb + hh;
        if (n_split_s == 1 && !TS_SPLIT_KEEP) {
            // hdr is a multiple of 8: a float4 of dims lies wholly inside or outside the row
            if (d < hdr) {
                const float inv = lsum > 0.0f ? 1.0f / lsum : 0.0f;
                const floatx4 r = lsum > 0.0f ? acc * inv : (floatx4)0.0f;
                *reinterpret_cast<float4 *>(a.out + head * hdr + d) = make_float4(r[0], r[1], r[2], r[3]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) store_partial(a, head, split, HD, d + k, acc[k], M, lsum);
        }
    }
    // without a split this is the launch's last kernel: it advances the lengths itself
    if (a.n_split == 1) arrive_and_advance(a);
