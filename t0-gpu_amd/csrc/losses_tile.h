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
__device__ __forceinline__ float row16_max(float v) {
    v = __builtin_fmaxf(v, dpp_row<0x128>(v));
    v = __builtin_fmaxf(v, dpp_row<0x124>(v));
    v = __builtin_fmaxf(v, dpp_row<0x122>(v));
    return __builtin_fmaxf(v, dpp_row<0x121>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_row<0x128>(v);
    v += dpp_row<0x124>(v);
    v += dpp_row<0x122>(v);
    return v + dpp_row<0x121>(v);
}

// e = 2^(u - m) is in [0, 2): no sign and a top exponent bit of 0, so 16 bits hold 7 of
// exponent and 9 of mantissa (rounded to nearest; relative error 2^-10, a quarter of
// bf16's).  A NaN does not survive, but its row's sum is NaN and scales every e.
__device__ __forceinline__ uint32_t pack_e(float lo, float hi) {
    const uint32_t a = (__builtin_bit_cast(uint32_t, lo) + 0x2000u) >> 14, b = (__builtin_bit_cast(uint32_t, hi) + 0x2000u) << 2;
    return (a & 0xFFFFu) | (b & 0xFFFF0000u);
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

// Element `reg` (0..3, uniform) of sub-tile `sub` = 8 i + j (uniform) of the accumulators, whose
// AGPRs can only be named: a binary tree of uniform branches.
template <int LO, int HI, int SM, int SN>
__device__ __forceinline__ float acc_pick(const f32x4_t (&acc)[SM][SN], uint32_t sub, uint32_t reg) {
    if constexpr (HI - LO == 1) {
        constexpr int I = LO / SN, J = LO % SN;
        const float a = acc_read(acc[I][J][0]), b = acc_read(acc[I][J][1]), c = acc_read(acc[I][J][2]),
                    d = acc_read(acc[I][J][3]);
        return reg < 2 ? (reg == 0 ? a : b) : (reg == 2 ? c : d);
    } else {
        constexpr int MID = (LO + HI) / 2;
        return sub < MID ? acc_pick<LO, MID>(acc, sub, reg) : acc_pick<MID, HI>(acc, sub, reg);
    }
}

// The raw logits of the entries (sorted tokens of each row) in a wave's 128 x 128 tile.  A
// lane looks at two rows; each hit is taken by the whole wave, from the lane that holds it.
template <int SM, int SN>
__device__ __forceinline__ void pick_entries(const T0gLossGemmArgs& a, const f32x4_t (&acc)[SM][SN], uint32_t row0,
                                             uint32_t col0, uint32_t lane) {
    const uint32_t width = col0 < a.g.n ? min(a.g.n - col0, T0G_LOSS_BLOCK) : 0u, first = a.v0 + col0;
#pragma unroll 1
    for (uint32_t half = 0; half < 2; ++half) {
        const uint32_t row = row0 + 64u * half + lane;
        uint32_t lo = 0, hi = 0;
        if (row < a.g.m) {
            hi = 1;
            if (a.ent_off) {
                const uint64_t o = (uint64_t)row * a.off_ld + first / T0G_LOSS_BLOCK;
                lo = *at<const uint16_t>(a.ent_off, o);
                hi = *at<const uint16_t>(a.ent_off, o + 1);
            }
        }
        for (;;) {
            uint32_t c = kNoToken;
            if (lo < hi) c = *at<const uint32_t>(a.ent_tok, (uint64_t)row * a.slots + lo) - first;
            uint64_t hits = __ballot(c < width);
            while (hits) {
                const uint32_t b = (uint32_t)__builtin_ctzll(hits);
                hits &= hits - 1;
                const uint32_t col = (uint32_t)__builtin_amdgcn_readlane((int)c, (int)b);
                const uint32_t slot = (uint32_t)__builtin_amdgcn_readlane((int)lo, (int)b);
                const uint32_t rr = 64u * half + b;
                const float z = acc_pick<0, SM * SN>(acc, (rr >> 4) * SN + (col >> 4), rr & 3u);
                if (lane == (((rr >> 2) & 3u) << 4 | (col & 15u)))
                    *at<float>(a.ent_z, (uint64_t)(row0 + rr) * a.slots + slot) = z;
            }
            ++lo;
            if (__ballot(lo < hi) == 0) break;
        }
    }
}

// Statistics of a wave's tile, per row over its 128 columns; KEEP: the exponentials go out
// in 16 bits.  Bound by v_exp_f32 (256 per lane, a quarter of the VALU's rate).
template <bool KEEP, int SM, int SN>
__device__ __forceinline__ void tile_stats(const T0gLossGemmArgs& a, const f32x4_t (&acc)[SM][SN], uint32_t row0,
                                           uint32_t col0, uint32_t lane, uint32_t lds) {
    asm volatile("v_mov_b32 %0, %0" : "+v"(lane));   // nothing below is hoisted above the K loop
    const uint32_t l16 = lane & 15u, q = lane >> 4;
    const uint32_t width = col0 < a.g.n ? min(a.g.n - col0, T0G_LOSS_BLOCK) : 0u;
    const uint64_t out = (uint64_t)(col0 / T0G_LOSS_BLOCK) * a.g.m;
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        __builtin_amdgcn_sched_barrier(0);   // one band at a time
        float z[SN][4], m[4], s[4], s2[4];
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
            for (int j = 1; j < SN; ++j) m[r] = __builtin_fmaxf(m[r], z[j][r]);
            m[r] = row16_max(m[r]) * a.k;
            m[r] = width ? m[r] : 0.0f;   // no columns: every exponential below is 2^-inf
            s[r] = s2[r] = 0.0f;
        }
        if (a.flags & T0G_LOSS_DUAL) {
            const float k2 = a.k * a.r;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < SN; ++j) s2[r] += exp2_(__builtin_fmaf(z[j][r], k2, -(m[r] * a.r)));
#pragma unroll
            for (int r = 0; r < 4; ++r) s2[r] = row16_sum(s2[r]);
        }
#pragma unroll
        for (int j = 0; j < SN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                z[j][r] = exp2_(__builtin_fmaf(z[j][r], a.k, -m[r]));
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
    }
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
    const uint32_t a_bytes = ((p.m - 1) * p.lda + p.k) * 2;
    const uint32_t b_bytes = (B_K ? (p.n - 1) * p.ldb + p.k : (p.k - 1) * p.ldb + p.n) * 2;
    const uint32_t lane = tid & 63u, wave = tid >> 6, wm = wave / 2, wn = wave % 2;
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
        const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
        Prefetch16 pf;
        pf.off = w < 2 ? prefetch_line<true>(m0, p.lda, cols, (n0 / BN) % cols, w & 1u, lane)
                       : prefetch_line<B_K>(n0, p.ldb, rows, (m0 / BM) % rows, w & 1u, lane);
        pf.base = w < 2 ? p.a : p.b;
        pf.bytes = w < 2 ? a_bytes : b_bytes;
        pf.kstep = 2u * (w < 2 || B_K ? 1u : p.ldb);
        k_pipeline16<false, A_BYTES, STAGE, kVmemPerStage, true>(acc, la, lb, p, a_bytes, b_bytes, 0, p.k, nst, lds0, pf);
    } else {
        k_pipeline16<false, A_BYTES, STAGE, kVmemPerStage>(acc, la, lb, p, a_bytes, b_bytes, 0, p.k, nst, lds0);
    }
    static_assert(2 * SN * 512 * (NT / 64) <= 2 * STAGE, "the staged bands fit");
    mfma16_drain();
    T0G_WAIT_VMCNT(0);
    barrier_no_fence();
    const uint32_t row0 = m0 + wm * WT, col0 = n0 + wn * WT, lds = lds_addr(smem) + wave * (2 * SN * 512);
    if constexpr (KIND == LossTile::Grad) {
        tile_grad(a, acc, row0, col0, lane, lds);
    } else {
        tile_stats<KIND == LossTile::Keep>(a, acc, row0, col0, lane, lds);
        pick_entries(a, acc, row0, col0, lane);
    }
}

}  // namespace t0g

#endif
