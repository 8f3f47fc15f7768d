// 256x256 GEMM tiles of the logits z = x W^T with the softmax in the epilogue, so that a
// large projection's logits never reach memory.  The K loop is the GEMM kernels'
// (gemm_mfma16.h: 4 waves of 128x128, one per SIMD).  Lane (q, c) of a wave holds, in
// sub-tile (i, j), rows 16 i + 4 q + 0..3 of column 16 j + c, so one row's 128 columns
// are 8 registers of 16 lanes.
#ifndef T0G_LOSSES_TILE_H
#define T0G_LOSSES_TILE_H

namespace t0g {

// Over the 16 lanes of a DPP row: rotations by 8, 4, 2 and 1 leave the result in all of them.
template <int CTRL>
__device__ __forceinline__ float dpp_row(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// (maximum, which passes NaN on, is one instruction; fmax quiets its operands first.)
__device__ __forceinline__ float max_(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float row16_max(float v) {
    v = max_(v, dpp_row<0x128>(v));
    v = max_(v, dpp_row<0x124>(v));
    v = max_(v, dpp_row<0x122>(v));
    return max_(v, dpp_row<0x121>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_row<0x128>(v);
    v += dpp_row<0x124>(v);
    v += dpp_row<0x122>(v);
    return v + dpp_row<0x121>(v);
}

// e = 2^(u - m) is in [0, 2): no sign and a top exponent bit of 0, so 16 bits hold 7 of
// exponent and 9 of mantissa, two more than bf16's.  They are cut off, not rounded: e is
// formed larger by the factor 1 + 2^-10 / (2 ln 2), what cutting takes off in the mean, which
// leaves a relative error of 0.7 2^-9 at most and none on average.  The factor costs
// nothing: its logarithm is subtracted from m.  A NaN does not survive, but its row's
// sum is NaN and scales every e.
constexpr float kKeepLog2 = 0.00101594f;
__device__ __forceinline__ uint32_t pack_e(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi) << 2, __builtin_bit_cast(uint32_t, lo) << 2, 0x07060302u);
}

// One 16-row band of a wave's sub-tiles, packed in 16 bits (w[j]: the lane's 4 rows of
// column 16 j + c), through LDS to 16-byte stores of whole lines, as store_tile_bf16_tr
// does.  `c`: address of the wave tile's first element, rows ldc apart.
template <int SN>
__device__ __forceinline__ void store_band16(const uint64_t (&w)[SN], uint64_t c, uint32_t ldc, int i, uint32_t lane,
                                             uint32_t lds) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    typedef __attribute__((address_space(3))) uint64_t lds_u64;
    const uint32_t reg = lds + (uint32_t)(i & 1) * (SN * 16 * 32);
    const uint32_t l16 = lane & 15u, q = lane >> 4, r = (lane >> 2) & 3u, s = lane & 3u;
#pragma unroll
    for (int j = 0; j < SN; ++j) *reinterpret_cast<lds_u64*>((uintptr_t)(reg + bf16_stage_off(16u * j + l16, q))) = w[j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const uint32_t rcol = 16u * q + 8u * (s & 1u) + r, rpc = s >> 1;
    const uint32_t srow = 4u * ((l16 >> 2) >> 1) + s, scol = 16u * q + 8u * ((l16 >> 2) & 1u);
    const uint64_t cb = c + ((uint64_t)srow * ldc + scol) * 2u;
#pragma unroll
    for (int u = 0; u < SN / 4; ++u)
#pragma unroll
        for (int pp = 0; pp < 2; ++pp) {
            const uint32_t c0 = 64u * u + rcol, piece = 2u * pp + rpc;
            const v4s lo =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(uintptr_t)(reg + bf16_stage_off(c0, piece)));
            const v4s hi =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(uintptr_t)(reg + bf16_stage_off(c0 + 4u, piece)));
            u32x4_t v;
            v[0] = __builtin_bit_cast(uint32_t, __builtin_shufflevector(lo, lo, 0, 1));
            v[1] = __builtin_bit_cast(uint32_t, __builtin_shufflevector(lo, lo, 2, 3));
            v[2] = __builtin_bit_cast(uint32_t, __builtin_shufflevector(hi, hi, 0, 1));
            v[3] = __builtin_bit_cast(uint32_t, __builtin_shufflevector(hi, hi, 2, 3));
            const uint64_t addr = cb + ((uint64_t)(16u * i + 8u * pp) * ldc + 64u * u) * 2u;
            __builtin_nontemporal_store(v, reinterpret_cast<__attribute__((address_space(1))) u32x4_t*>((uintptr_t)addr));
        }
}

// The raw logits of the entries (sorted tokens of each row) in a wave's 128 x 128 tile.
// Lane l looks after rows l and 64 + l.  Which entries a row has there, and its first two
// tokens, are loaded two bands of statistics ahead of their use, which covers the
// latency.  A 16-row band with any entry goes to LDS, [4-row quad][column][row in quad],
// from where the 16 lanes of its rows take what they need.  Taking each entry from the
// accumulators instead, through a tree of uniform branches, cost 13 us a tile with 64
// entries a row over 32000 tokens, as much as a quarter of the K loop at K = 2048.
struct EntryScan {
    uint32_t range[2];      // entries before the block and before the next (u16 each)
    uint32_t tok[2][2];
};

__device__ __forceinline__ void scan_ranges(const T0gLossGemmArgs& a, EntryScan& e, uint32_t row0, uint32_t col0,
                                            uint32_t lane) {
    typedef uint32_t u32_2 __attribute__((aligned(2)));
    const uint32_t block = min((a.v0 + col0) / T0G_LOSS_BLOCK, a.off_ld - 2);   // a wave past the vocabulary takes none
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t row = row0 + 64u * h + lane;
        e.range[h] = 1u << 16;
        if (a.ent_off)
            e.range[h] = *reinterpret_cast<gptr<const u32_2>>(
                (uintptr_t)(a.ent_off + ((uint64_t)min(row, a.g.m - 1) * a.off_ld + block) * 2));
    }
}

__device__ __forceinline__ void scan_tokens(const T0gLossGemmArgs& a, EntryScan& e, uint32_t row0, uint32_t lane) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t row = row0 + 64u * h + lane;
        if (row >= a.g.m) e.range[h] = 0;
        const uint64_t slot = (uint64_t)min(row, a.g.m - 1) * a.slots;
        const uint32_t lo = e.range[h] & 0xFFFFu;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) e.tok[h][i] = *at<const uint32_t>(a.ent_tok, slot + min(lo + i, a.slots - 1));
    }
}

template <int I, int SM, int SN>
__device__ __forceinline__ void pick_band(const T0gLossGemmArgs& a, const f32x4_t (&acc)[SM][SN], const EntryScan& e,
                                          uint32_t row0, uint32_t col0, uint32_t lane, uint32_t lds) {
    typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;
    typedef const __attribute__((address_space(3))) float lds_f32;
    constexpr uint32_t H = I / 4;
    const uint32_t width = col0 < a.g.n ? min(a.g.n - col0, T0G_LOSS_BLOCK) : 0u, first = a.v0 + col0;
    const uint32_t lo = e.range[H] & 0xFFFFu, hi = e.range[H] >> 16;
    const bool mine = (lane >> 4) == I % 4 && lo < hi;
    // a row without an offset table has one slot, which may hold any token or none
    if (__ballot(mine && (a.ent_off || e.tok[H][0] - first < width)) == 0) return;
    const uint32_t l16 = lane & 15u, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < SN; ++j)
        *reinterpret_cast<lds_f32x4*>((uintptr_t)(lds + q * (SN * 256) + (16u * j + l16) * 16u)) =
            f32x4_t{acc_read(acc[I][j][0]), acc_read(acc[I][j][1]), acc_read(acc[I][j][2]), acc_read(acc[I][j][3])};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (mine) {
        const uint64_t slot = (uint64_t)(row0 + 64u * H + lane) * a.slots;
        const uint32_t base = lds + (l16 >> 2) * (SN * 256) + (l16 & 3u) * 4u;   // row 16 I + l16 of the tile
        for (uint32_t s = lo; s < hi; ++s) {
            const uint32_t t = s == lo ? e.tok[H][0] : s == lo + 1 ? e.tok[H][1] : *at<const uint32_t>(a.ent_tok, slot + s);
            const uint32_t c = t - first;
            if (c < width) *at<float>(a.ent_z, slot + s) = *reinterpret_cast<lds_f32*>((uintptr_t)(base + c * 16u));
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next band overwrites it
}

// Statistics of a wave's tile, per row over its 128 columns; KEEP: the exponentials go out
// in 16 bits.  Bound by v_exp_f32 (256 per lane, a quarter of the VALU's rate).
template <bool KEEP, int SM, int SN>
__device__ __forceinline__ void tile_stats(const T0gLossGemmArgs& a, const f32x4_t (&acc)[SM][SN], uint32_t row0,
                                           uint32_t col0, uint32_t lane, uint32_t lds, uint32_t pick_lds) {
    asm volatile("v_mov_b32 %0, %0" : "+v"(lane));   // nothing below is hoisted above the K loop
    EntryScan scan;
    scan_ranges(a, scan, row0, col0, lane);
    const uint32_t l16 = lane & 15u, q = lane >> 4;
    const uint32_t width = col0 < a.g.n ? min(a.g.n - col0, T0G_LOSS_BLOCK) : 0u;
    const uint64_t out = (uint64_t)(col0 / T0G_LOSS_BLOCK) * a.g.m;
    auto pick = [&](auto band) { pick_band<band.value>(a, acc, scan, row0, col0, lane, pick_lds); };
    auto stats = [&](int i) {
        __builtin_amdgcn_sched_barrier(0);   // one band at a time
        float z[SN][4], m[4], from[4], s[4], s2[4];
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[j][r] = acc_read(acc[i][j][r]);
        if (width < T0G_LOSS_BLOCK)
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[j][r] = 16u * j + l16 < width ? z[j][r] : ninf();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m[r] = z[0][r];
#pragma unroll
            for (int j = 1; j < SN; ++j) m[r] = max_(m[r], z[j][r]);
            m[r] = KEEP ? __builtin_fmaf(row16_max(m[r]), a.k, -kKeepLog2) : row16_max(m[r]) * a.k;
            m[r] = width ? m[r] : 0.0f;   // no columns: every exponential below is 2^-inf
            from[r] = m[r] == ninf() ? 0.0f : m[r];   // no token left: sums of 0, not of 2^(-inf + inf)
            s[r] = s2[r] = 0.0f;
        }
        if (a.flags & T0G_LOSS_DUAL) {
            const float k2 = a.k * a.r;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < SN; ++j) s2[r] += exp2_(__builtin_fmaf(z[j][r], k2, -(from[r] * a.r)));
#pragma unroll
            for (int r = 0; r < 4; ++r) s2[r] = row16_sum(s2[r]);
        }
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                z[j][r] = exp2_(__builtin_fmaf(z[j][r], a.k, -from[r]));
                s[r] += z[j][r];
            }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = row16_sum(s[r]);
        if constexpr (KEEP) {
            uint64_t w[SN];
#pragma unroll
            for (int j = 0; j < SN; ++j)
                w[j] = pack_e(z[j][0], z[j][1]) | (uint64_t)pack_e(z[j][2], z[j][3]) << 32;
            store_band16<SN>(w, a.g.c + ((uint64_t)row0 * a.g.ldc + col0) * 2, a.g.ldc, i, lane, lds);
        }
        // lane c < 4 of each row of lanes stores row 4 q + c
        const float ms = l16 < 2 ? (l16 == 0 ? m[0] : m[1]) : (l16 == 2 ? m[2] : m[3]);
        const float ss = l16 < 2 ? (l16 == 0 ? s[0] : s[1]) : (l16 == 2 ? s[2] : s[3]);
        const uint32_t row = row0 + 16u * i + 4u * q + l16;
        if (l16 < 4 && row < a.g.m && width) {
            *at<f32x2_t>(a.part, out + row) = f32x2_t{ms, ss};
            if (a.flags & T0G_LOSS_DUAL)
                *at<float>(a.part2, out + row) = l16 < 2 ? (l16 == 0 ? s2[0] : s2[1]) : (l16 == 2 ? s2[2] : s2[3]);
        }
    };
    static_assert(SM == 8, "eight bands");
    stats(0);
    scan_tokens(a, scan, row0, lane);
    stats(1);
    stats(2);
    pick(std::integral_constant<int, 0>{});
    stats(3);
    pick(std::integral_constant<int, 1>{});
    stats(4);
    pick(std::integral_constant<int, 2>{});
    stats(5);
    pick(std::integral_constant<int, 3>{});
    stats(6);
    pick(std::integral_constant<int, 4>{});
    stats(7);
    pick(std::integral_constant<int, 5>{});
    pick(std::integral_constant<int, 6>{});
    pick(std::integral_constant<int, 7>{});
}

// The dense part of the logits' gradients, zero past the piece's columns and rows.
template <int SM, int SN>
__device__ __forceinline__ void tile_grad(const T0gLossGemmArgs& a, const f32x4_t (&acc)[SM][SN], uint32_t row0,
                                          uint32_t col0, uint32_t lane, uint32_t lds) {
    asm volatile("v_mov_b32 %0, %0" : "+v"(lane));
    const uint32_t l16 = lane & 15u, q = lane >> 4;
    const uint32_t width = col0 < a.g.n ? min(a.g.n - col0, T0G_LOSS_BLOCK) : 0u;
    const float k2 = a.k * a.r;
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t par[4];
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t row = row0 + 16u * i + 4u * q + r;
            par[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (row < a.g.m) par[r] = *at<const f32x4_t>(a.row_par, row);
        }
        float z[SN][4];
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[j][r] = acc_read(acc[i][j][r]);
        if (a.flags & T0G_LOSS_DUAL) {
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    z[j][r] = __builtin_fmaf(par[r][2], exp2_(__builtin_fmaf(z[j][r], a.k, -par[r][0])),
                                             par[r][3] * exp2_(__builtin_fmaf(z[j][r], k2, -par[r][1])));
        } else {
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[j][r] = par[r][2] * exp2_(__builtin_fmaf(z[j][r], a.k, -par[r][0]));
        }
        if (width < T0G_LOSS_BLOCK)
#pragma unroll
            for (int j = 0; j < SN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) z[j][r] = 16u * j + l16 < width ? z[j][r] : 0.0f;
        uint64_t w[SN];
#pragma unroll
        for (int j = 0; j < SN; ++j) w[j] = pack2(z[j][0], z[j][1]) | (uint64_t)pack2(z[j][2], z[j][3]) << 32;
        store_band16<SN>(w, a.g.c + ((uint64_t)row0 * a.g.ldc + col0) * 2, a.g.ldc, i, lane, lds);
    }
}

enum class LossTile { Stats, Keep, Grad };

template <bool B_K, LossTile KIND>
__device__ __forceinline__ void loss_tile(const T0gLossGemmArgs& a) {
    const T0gGemmArgs& p = a.g;
    constexpr int BM = 256, BN = 256, NT = 256, WT = 128, SM = WT / 16, SN = WT / 16;
    using OpA = Op16<true, BM, NT, SM>;
    using OpB = Op16<B_K, BN, NT, SN>;
    constexpr uint32_t A_BYTES = OpA::kStageBytes, STAGE = OpA::kStageBytes + OpB::kStageBytes;
    constexpr int kVmemPerStage = OpA::kInstr + OpB::kInstr;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    const uint32_t tid = threadIdx.x;
    uint32_t m0, n0;
    tile_origin<BM, BN>(p, m0, n0);
    const int nst = (int)((p.k + 63) / 64);
    const uint32_t a_bytes = operand_bytes<true>(p.m, p.k, p.lda), b_bytes = operand_bytes<B_K>(p.n, p.k, p.ldb);
    const uint32_t lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / 2, wn = wave % 2;
    OpA la;
    OpB lb;
    la.init(tid, m0, p.lda, wm * WT);
    lb.init(tid, n0, p.ldb, wn * WT);
    f32x4_t acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) acc[i][j] = f32x4_t{};
    mfma16_drain();
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    if (p.k % 64 != 0) {
        k_pipeline16<true, A_BYTES, STAGE, kVmemPerStage>(acc, la, lb, p, a_bytes, b_bytes, 0, p.k, nst, lds0);
    } else if (p.flags & T0G_FLAG_PREFETCH) {
        const uint32_t rows = p.tiles_m >= 8 ? 8u : p.tiles_m >= 4 ? 4u : 2u, cols = rows == 8 ? 4u : 8u;
        Prefetch16 pf;
        pf.off = wave < 2 ? prefetch_line<true>(m0, p.lda, cols, (n0 / BN) % cols, wave & 1u, lane)
                          : prefetch_line<B_K>(n0, p.ldb, rows, (m0 / BM) % rows, wave & 1u, lane);
        pf.base = wave < 2 ? p.a : p.b;
        pf.bytes = wave < 2 ? a_bytes : b_bytes;
        pf.kstep = 2u * (wave < 2 || B_K ? 1u : p.ldb);
        k_pipeline16<false, A_BYTES, STAGE, kVmemPerStage, true>(acc, la, lb, p, a_bytes, b_bytes, 0, p.k, nst, lds0, pf);
    } else {
        k_pipeline16<false, A_BYTES, STAGE, kVmemPerStage>(acc, la, lb, p, a_bytes, b_bytes, 0, p.k, nst, lds0);
    }
    constexpr uint32_t kBands = 2 * SN * 512, kPick = SN * 1024;   // LDS of a wave: two bands in 16 bits, one in f32
    static_assert((kBands + kPick) * (NT / 64) <= 2 * STAGE, "the staged bands fit");
    mfma16_drain();
    T0G_WAIT_VMCNT(0);
    barrier_no_fence();
    const uint32_t row0 = m0 + wm * WT, col0 = n0 + wn * WT, lds = lds_addr(smem) + wave * kBands;
    if constexpr (KIND == LossTile::Grad) {
        tile_grad(a, acc, row0, col0, lane, lds);
    } else {
        tile_stats<KIND == LossTile::Keep>(a, acc, row0, col0, lane, lds, lds_addr(smem) + 4 * kBands + wave * kPick);
    }
}

}  // namespace t0g

#endif
