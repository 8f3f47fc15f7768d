// The gated pair of products in 256x256 tiles of the GEMM kernels' K loop (gemm_mfma16.h: 4 waves of 128x128, one per
// SIMD): 128 features of both weights, in the order 64 of Wg, 64 of Wu, 64 of Wg, 64 of Wu, so that a wave holds
// g (sub-tiles 0 to 3 of a row of them) and u (4 to 7) of the same 64 features.  Bound, as these kernels are, by
// the clock that the board's power allows.
#ifndef T0G_FFN_GATED_H
#define T0G_FFN_GATED_H

namespace t0g {

// [features][ld]: every request's 8 rows are of one weight, and of the same one for a wave.
struct PairK : Op16<true, 256, 256, 8> {
    uint64_t own;
    __device__ __forceinline__ void init_pair(const T0gTileArgs& p, uint32_t tid, uint32_t n0, uint32_t wrow) {
        init(tid, 0, p.ldb, wrow);
        const uint32_t lane = tid & 63u;
        own = wave & 1u ? p.b2 : p.b;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const uint32_t r = 8 * i + (lane >> 3), c = (lane & 7u) ^ fk<64>(r);   // fk: 64-row steps do not matter
            offs[i] = ((n0 + 64 * (wave >> 1) + r) * p.ldb + c * 8) * 2 - (uint32_t)(i & 3) * 1024u;
        }
    }
    __device__ __forceinline__ u32x4_t rsrc(uint64_t, uint32_t bytes, uint32_t, uint32_t k0) const {
        return rsrc_words32(own, bytes, k0 * 2);
    }
    template <bool CHECK>
    __device__ __forceinline__ void issue_one(int i, u32x4_t r, uint32_t lds, uint32_t k0, uint32_t kend) const {
        if (CHECK) {
            const uint32_t lane = threadIdx.x & 63u, kc = 8 * ((lane & 7u) ^ fk<64>(8 * i + (lane >> 3)));
            dma16(r, k0 + kc < kend ? offs[i] + (uint32_t)(i & 3) * 1024u : kOob, lds + (wave * kInstr + i) * 1024);
        } else {
            if ((i & 3) == 0) dma_m0(lds, (wave * kInstr + i) * 1024);
            dma16_slot(r, offs[i], i & 3);
        }
    }
    template <bool CHECK>
    __device__ __forceinline__ void issue(uint32_t lds, uint64_t base, uint32_t bytes, uint32_t ld, uint32_t k0, uint32_t kend) const {
        const u32x4_t r = rsrc(base, bytes, ld, k0);
#pragma unroll
        for (int i = 0; i < kInstr; ++i) issue_one<CHECK>(i, r, lds, k0, kend);
    }
};

// [k][ld]: a request is two rows of k of the tile's 256 columns, of both weights, which the host
// lays within 2 GiB of each other; p.b is the one that comes first.
struct PairN : Op16<false, 256, 256, 8> {
    __device__ __forceinline__ void init_pair(const T0gTileArgs& p, uint32_t tid, uint32_t n0, uint32_t wrow) {
        init(tid, 0, p.ldb, wrow);
        const uint32_t lane = tid & 63u;
        const uint64_t first = p.b < p.b2 ? p.b : p.b2;
        const uint32_t to[2] = {(uint32_t)(p.b - first), (uint32_t)(p.b2 - first)};
        const uint32_t slot = lane & 31u;
        auto at_ = [&](uint32_t k) {   // byte offset of the lane's piece of row k of a stage
            const uint32_t g = (slot >> 1) ^ fm16(k, kGranules), f = n0 + (g >> 3) * 64 + (g & 3u) * 16 + (slot & 1u) * 8;
            // past the features the first weight's rows are not bounded by the descriptor
            return f < p.n ? (g >> 2 & 1u ? to[1] : to[0]) + (k * p.ldb + f) * 2 : kOob;
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) off[i] = at_(2 * wave + (lane >> 5) + 2 * kWaves * i) - i * step;
#pragma unroll
        for (int i = 0; i < kInstr; ++i) offs[i] = at_(2 * (wave * kInstr + i) + (lane >> 5)) - (uint32_t)(i & 3) * 1024u;
    }
};

template <bool NC>
__device__ __forceinline__ void gated_big(const T0gTileArgs& p) {
    constexpr int BM = 256, NT = 256, SM = 8, SN = 8;
    using OpA = Op16<true, BM, NT, SM>;
    using OpB = typename std::conditional<NC, PairN, PairK>::type;
    constexpr uint32_t A_BYTES = OpA::kStageBytes, STAGE = OpA::kStageBytes + OpB::kStageBytes;
    constexpr int kVmemPerStage = OpA::kInstr + OpB::kInstr;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    const uint32_t tid = threadIdx.x;
    uint32_t tm, tn;
    tile_of(p, tm, tn);
    const uint32_t m0 = tm * BM, n0 = tn * 128, k8 = (p.k + 7) & ~7u;
    T0gGemmArgs g;
    g.a = p.a;
    g.b = p.b < p.b2 ? p.b : p.b2;
    g.lda = p.lda;
    g.ldb = p.ldb;
    const uint32_t a_bytes = operand_bytes<true>(p.m, k8, p.lda);
    uint32_t b_bytes;
    if constexpr (NC)
        b_bytes = operand_bytes<false>(p.n, p.k, p.ldb) + (uint32_t)(p.b < p.b2 ? p.b2 - p.b : p.b - p.b2);
    else
        b_bytes = operand_bytes<true>(p.n, k8, p.ldb);
    const uint32_t lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / 2, wn = wave % 2;
    OpA la;
    OpB lb;
    la.init(tid, m0, p.lda, wm * 128);
    lb.init_pair(p, tid, n0, wn * 128);
    f32x4_t acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) acc[i][j] = f32x4_t{};
    mfma16_drain();
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    const int nst = (int)((p.k + 63) / 64);
    if (p.k % 64 != 0)
        k_pipeline16<true, A_BYTES, STAGE, kVmemPerStage>(acc, la, lb, g, a_bytes, b_bytes, 0, p.k, nst, lds0);
    else
        k_pipeline16<false, A_BYTES, STAGE, kVmemPerStage>(acc, la, lb, g, a_bytes, b_bytes, 0, p.k, nst, lds0);
    mfma16_drain();
    T0G_WAIT_VMCNT(0);
    barrier_no_fence();
    const uint32_t row0 = m0 + wm * 128, col0 = n0 + wn * 64, l16 = lane & 15u, q = lane >> 4, lds = lds_addr(smem) + wave * 4096;
    // whole waves of aligned rows leave in 16-byte pieces through LDS
    const bool whole = row0 + 128 <= p.m && col0 + 64 <= p.n && !(p.flags & T0G_TILE_OUT_F32) && p.ldc % 8 == 0 && p.c % 16 == 0 &&
                       (!(p.gate || p.up) || (p.ldg % 8 == 0 && p.gate % 16 == 0 && p.up % 16 == 0));
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        __builtin_amdgcn_sched_barrier(0);   // one band at a time
        float h[4][4], gv[4][4], uv[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                gv[j][r] = acc_read(acc[i][j][r]);
                uv[j][r] = acc_read(acc[i][j + 4][r]);
                float a, slope;
                activation(p.act, gv[j][r], a, slope);
                h[j][r] = a * uv[j][r];
            }
        auto band = [&](uint64_t to, uint32_t ld, const float (&v)[4][4], bool f32) {
            if (whole) {
                uint64_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pack2(v[j][0], v[j][1]) | (uint64_t)pack2(v[j][2], v[j][3]) << 32;
                store_band16<4>(w, to + ((uint64_t)row0 * ld + col0) * 2, ld, i, lane, lds);
                return;
            }
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t row = row0 + 16 * i + 4 * q + r;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t col = col0 + 16 * j + l16;
                    if (row < p.m && col < p.n) {
                        if (f32)
                            *at<float>(to, (uint64_t)row * ld + col) = v[j][r];
                        else
                            *at<__bf16>(to, (uint64_t)row * ld + col) = (__bf16)v[j][r];
                    }
                }
            }
        };
        band(p.c, p.ldc, h, p.flags & T0G_TILE_OUT_F32);
        if (p.gate) band(p.gate, p.ldg, gv, false);
        if (p.up) band(p.up, p.ldg, uv, false);
    }
}

}  // namespace t0g

#endif
