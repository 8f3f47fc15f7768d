// The 256 x 256 tile of the 8-bit product with a bf16 result: 8 waves of 128 x 64, two on a SIMD, two 66 KB
// stages of 128 K values.
#ifndef T0G_FFN_BIG_H
#define T0G_FFN_BIG_H

namespace t0g {

template <int FA, int FB, bool B_TILE>
__device__ __forceinline__ void f8_big(const T0gTileArgs& p) {
    constexpr int BM = 256, BN = 256, W = 8, WN = 4, TM = 128, TN = 64, SM = TM / 16, SN = TN / 16;
    using OpA = RowsK<BM, W>;
    using OpB = RowsK<BN, W>;
    constexpr uint32_t A = OpA::kBytes, AB = A + OpB::kBytes, STAGE = AB + (BM + BN) * 4;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN, l16 = lane & 15u, q = lane >> 4;
    uint32_t tm, tn;
    tile_of(p, tm, tn);
    const uint32_t m0 = tm * BM, n0 = tn * BN, kb = (p.k + 15) & ~15u;
    OpA la;
    OpB lb;
    la.init(p.a, m0, p.m, p.lda, kb, wave, lane, wm * TM);
    lb.init(p.b, n0, p.n, p.ldb, kb, wave, lane, wn * TN);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    const uint32_t nst = (p.k + 127) / 128;
    f32x4_t acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // A stage past the end brings zeros and reads no memory.  Scales, 64 a request: waves 0 to 3 bring A's, 4 to 7 B's.
    const bool mine = wave < 4;
    const uint32_t at64 = 64 * (wave & 3u) + lane;   // a scale for each 128 columns is spread to the columns
    const uint64_t sbase = mine ? p.as : p.bs, sld = (uint64_t)(mine ? p.ldas : p.ldbs) * 4;
    const uint64_t sbytes = (uint64_t)(mine ? p.m : B_TILE ? (p.n + 127) / 128 : p.n) * 4;
    const uint32_t soff = (mine ? m0 + at64 : B_TILE ? (n0 + at64) / 128 : n0 + at64) * 4;
    auto issue_scales = [&](uint32_t s, uint32_t lds) {
        const u32x4_t r = rsrc_words_wide(sbase, (s < nst ? sbytes : 0u) + (uint64_t)s * sld, (uint64_t)s * sld);
        dma4(r, soff, lds + AB + 256 * wave);
    };
    typedef const __attribute__((address_space(3))) f32x4_t lds_f32x4;
    typedef const __attribute__((address_space(3))) float lds_f32;
    i32x8_t fb[SN], fa[3];
    f32x4_t sbv[B_TILE ? 1 : SN];
    float sa[3];
    const uint32_t sa_at = AB + (wm * TM + l16) * 4, sb_at = AB + (BM + wn * TN + 4 * q) * 4;   // offsets of the lane's scales
    auto read_a = [&](uint32_t stage, int i, int to) {
        fa[to] = join(la.template read<0>(stage, i), la.template read<1>(stage, i));
        sa[to] = reinterpret_cast<lds_f32*>((uintptr_t)(stage + sa_at))[16 * i];
    };
    auto read_b = [&](uint32_t stage, int j) { fb[j] = join(lb.template read<0>(stage + A, j), lb.template read<1>(stage + A, j)); };
    auto read_sb = [&](uint32_t stage, int j) {
        if constexpr (!B_TILE) sbv[j] = reinterpret_cast<lds_f32x4*>((uintptr_t)(stage + sb_at))[4 * j];
    };
    la.issue(lds0, 0, kb, wave);
    lb.issue(lds0 + A, 0, kb, wave);
    issue_scales(0, lds0);
    T0G_WAIT_VMCNT(0);
    barrier_no_fence();
    la.issue(lds0 + STAGE, 128, kb, wave);
    read_a(lds0, 0, 0);
#pragma unroll
    for (int j = 0; j < SN; ++j) read_b(lds0, j);
    uint32_t cur = lds0;
    // Matrix instruction t and, beside it, the vector instructions on the result of t - kBehind and a read for
    // a row of sub-tiles to come, pinned in this order: the compiler's own puts each result's use right
    // behind it, where the wave waits for it.  The last two rows of sub-tiles go column by column, so that
    // B's fragments of the next stage follow into the registers of this one's: at the stage's
    // start all waves would read them at once and the matrix units wait for LDS.  Before these rows the
    // waves meet: the next stage is there, and this one's fragments are all in registers, so the stage
    // after next starts on its way into their place.
    constexpr int kBehind = 3, T = SM * SN, kLast = T - 2 * SN;
    static_assert(2 * OpA::kInstr <= 2 * SN && 2 * OpB::kInstr < kLast, "a stage's requests fit");
    for (uint32_t s = 0; s < nst; ++s) {
        const uint32_t nxt = lds0 + (cur == lds0 ? STAGE : 0u);
        // (through LDS: a load of the compiler's would be waited for together with all DMA before it)
        float sbc = 0.0f;
        if constexpr (B_TILE) sbc = *reinterpret_cast<lds_f32*>((uintptr_t)(cur + AB + (BM + wn * TN) * 4));
#pragma unroll
        for (int j = 0; j < SN; ++j) read_sb(cur, j);
        const u32x4_t rb = lb.rsrc((s + 1) * 128), ra = la.rsrc((s + 2) * 128);
        f32x4_t v[kBehind + 1];
        float f[SM];
        auto row_of = [](int t) { return t < kLast ? t / SN : SM - 2 + (t - kLast) % 2; };
        // a row's fragment registers: rows next to each other, the last three, and the next stage's first beside the last
        // two have different ones
        auto slot_of = [](int i) { return i == 2 || i == SM - 1 ? 2 : i == 1 || i == 4 || i == SM - 2 ? 1 : 0; };
        auto col_of = [](int t) { return t < kLast ? t % SN : (t - kLast) / 2; };
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < T + kBehind; ++t) {
            if (t == kLast) {
                __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0): the next stage is there; lgkmcnt(0): this one is read
                barrier_no_fence();
                __builtin_amdgcn_sched_barrier(0);
            }
            if (t < T) {
                const int i = row_of(t), j = col_of(t);
                if (j == 0) f[i] = B_TILE ? sa[slot_of(i)] * sbc : sa[slot_of(i)];
                v[t % (kBehind + 1)] = mfma_f8<FB, FA>(fb[j], fa[slot_of(i)], f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                if (t < kLast) {
                    if (j == 0 && i < SM - 2) read_a(cur, i + 1, slot_of(i + 1));
                    if (j == 1 && i == SM - 3) read_a(cur, SM - 1, slot_of(SM - 1));
                } else if (i == SM - 1) {
                    read_b(nxt, j);
                    if (j == 0) read_a(nxt, 0, 0);
                }
            }
            // the stage's DMA, a request every other matrix instruction: B's half of the next one, A's of that after
            if (t < 2 * OpB::kInstr && t % 2 == 1) lb.issue_one(t / 2, rb, nxt + A, (s + 1) * 128, kb, wave);
            if (t == 2 * OpB::kInstr) issue_scales(s + 1, nxt);
            if (t >= kLast && t < T && t % 2 == 1) la.issue_one((t - kLast) / 2, ra, cur, (s + 2) * 128, kb, wave);
            if (t >= kBehind) {
                const int o = t - kBehind, oi = row_of(o), oj = col_of(o);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = v[o % (kBehind + 1)][e];
                    acc[oi][oj][e] = __builtin_fmaf(B_TILE ? x : x * sbv[B_TILE ? 0 : oj][e], f[oi], acc[oi][oj][e]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        cur = nxt;
    }
    T0G_WAIT_VMCNT(0);   // stages past the end: the LDS is the next workgroup's
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        const uint32_t row = m0 + wm * TM + 16 * i + l16;
        if (row < p.m)
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                const uint32_t col = n0 + wn * TN + 16 * j + 4 * q;
                store4(p.c, (uint64_t)row * p.ldc + col, left4(p.n, col), false, acc[i][j]);
            }
    }
}

}  // namespace t0g

#endif
