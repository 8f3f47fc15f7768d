// Tile kernels of the feed-forward layer's products: C = A B^T of 8-bit values with block
// scales, and the gated pair of bf16 products.  Both stage 128 bytes of K of every row (128
// values of 8 bits, 64 of bf16) in LDS by DMA, NS stages in turn, and multiply 16x16
// sub-tiles with the operands swapped: the matrix unit's rows are C's columns, so lane
// (q, c) of a sub-tile holds columns 4 q .. 4 q + 3 of row c of C, neighbours in memory, and
// a row's scale is one register.
#ifndef T0G_FFN_TILE_H
#define T0G_FFN_TILE_H

namespace t0g {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

// 4-byte buffer loads straight into LDS: lane l's value goes to m0 + 4 l.
__device__ __forceinline__ void dma4(u32x4_t rsrc, uint32_t voff, uint32_t lds_m0) {
    asm volatile(
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "buffer_load_dword %0, %1, 0 offen lds"
        :
        : "v"(voff), "s"(rsrc), "s"(lds_m0)
        : "memory", "m0");
}

// The tile of this workgroup: workgroups go to the 8 XCDs in turn, so each XCD takes a
// contiguous share of the tiles, and of these group_m rows of tiles at a time, which share
// their panels in its L2.
__device__ __forceinline__ void tile_of(const T0gTileArgs& p, uint32_t& tm, uint32_t& tn) {
    const uint32_t total = p.tiles_m * p.tiles_n, x = blockIdx.x & 7u, per = total >> 3, more = total & 7u;
    const uint32_t id = x * per + min(x, more) + (blockIdx.x >> 3);
    const uint32_t band = p.group_m * p.tiles_n, first = id / band * p.group_m, in = id % band;
    const uint32_t high = min(p.group_m, p.tiles_m - first);
    tm = first + in % high;
    tn = in / high;
}

// K-contiguous operand, ROWS rows of 128 bytes a stage: 16-byte chunk c of row r at chunk
// c ^ (r / 2 % 8), which puts the 16 rows of a sub-tile on distinct banks.  One request brings 8 rows.
template <int ROWS, int W>
struct RowsK {
    static constexpr int kInstr = ROWS / 8 / W;
    static_assert(kInstr * 8 * W == ROWS && W % 2 == 0, "whole requests, the swizzle the same in all of a wave's");
    static constexpr uint32_t kBytes = ROWS * 128;
    uint64_t base, bytes;   // the tile's first row, and from there to the operand's end
    uint32_t off, step, kcol, frag;

    __device__ __forceinline__ void init(uint64_t operand, uint32_t row0, uint32_t rows, uint64_t ldb, uint32_t kb, uint32_t wave,
                                         uint32_t lane, uint32_t wrow) {
        const uint32_t r = 8 * wave + (lane >> 3), c = (lane & 7u) ^ ((r >> 1) & 7u), l16 = lane & 15u, q = lane >> 4;
        base = operand + (uint64_t)row0 * ldb;
        bytes = (uint64_t)(min(rows - row0, (uint32_t)ROWS) - 1) * ldb + kb;
        kcol = 16 * c;
        off = r * (uint32_t)ldb + kcol;
        step = 8 * W * (uint32_t)ldb;
        frag = (wrow + l16) * 128 + ((q ^ ((l16 >> 1) & 7u)) << 4);
    }
    // Stage at byte k0 of K, kb bytes in all.
    __device__ __forceinline__ u32x4_t rsrc(uint32_t k0) const { return rsrc_words_wide(base, bytes, k0); }
    __device__ __forceinline__ void issue_one(int i, u32x4_t r, uint32_t lds, uint32_t k0, uint32_t kb, uint32_t wave) const {
        dma16(r, k0 + kcol < kb ? off + i * step : kOob, lds + (i * W + wave) * 1024);
    }
    __device__ __forceinline__ void issue(uint32_t lds, uint32_t k0, uint32_t kb, uint32_t wave) const {
        const u32x4_t r = rsrc(k0);
#pragma unroll
        for (int i = 0; i < kInstr; ++i) issue_one(i, r, lds, k0, kb, wave);
    }
    // Chunks q and 4 + q of 16 rows: K values in an order of their own, the same for both operands.
    template <int HALF>
    __device__ __forceinline__ i32x4_t read(uint32_t stage, int sub) const {
        const __attribute__((address_space(3))) i32x4_t* a =
            reinterpret_cast<const __attribute__((address_space(3))) i32x4_t*>((uintptr_t)(stage + (frag ^ (HALF << 6))));
        return a[sub * 128];
    }
};

// N-contiguous bf16 operand [k][ld], COLS columns of 64 k rows a stage: 32-byte granule g of
// row k at granule g ^ fm16(k).
template <int COLS, int W>
struct RowsN {
    static constexpr uint32_t kRowB = COLS * 2, kGranules = COLS / 16, kBytes = 64 * kRowB;
    static constexpr int kInstr = kBytes / 1024 / W;
    static constexpr uint32_t kRows = 1024 / kRowB;   // k rows of a request
    static_assert(kInstr * 1024 * W == kBytes && kGranules >= 4, "whole requests");
    uint64_t base, bytes;
    uint32_t col, slot, frag, ld;

    __device__ __forceinline__ void init(uint64_t operand, uint32_t col0, uint32_t cols, uint32_t k, uint32_t ld_, uint32_t wave,
                                         uint32_t lane, uint32_t wcol) {
        ld = ld_;
        base = operand + (uint64_t)col0 * 2;
        bytes = ((uint64_t)(k - 1) * ld + (((cols + 7) & ~7u) - col0)) * 2;
        slot = lane % (kRowB / 16);
        const uint32_t q = lane >> 4, r = (lane >> 2) & 3u, c = lane & 3u, k0 = 8 * q + r;
        frag = k0 * kRowB + c * 8 + (((wcol >> 4) ^ fm16(k0, kGranules)) << 5);
        (void)wave;
    }
    __device__ __forceinline__ void issue(uint32_t lds, uint32_t k0, uint32_t k, uint32_t wave, uint32_t lane) const {
        const u32x4_t rs = rsrc_words_wide(base, bytes, (uint64_t)k0 * ld * 2);
#pragma unroll
        for (int i = 0; i < kInstr; ++i) {
            const uint32_t kr = (i * W + wave) * kRows + lane / (kRowB / 16);
            const uint32_t g = (slot >> 1) ^ fm16(kr, kGranules);
            dma16(rs, k0 + kr < k ? (kr * ld + g * 16 + (slot & 1u) * 8) * 2 : kOob, lds + (i * W + wave) * 1024);
        }
    }
    // Sub-tile granules are XORed: sub is below the wave's (a power of two) of them.
    template <int HALF>
    __device__ __forceinline__ i32x4_t read(uint32_t stage, int sub) const {
        constexpr int O0 = HALF * 32 * kRowB, O1 = (HALF * 32 + 4) * kRowB;
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef short v8s __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const __attribute__((address_space(3))) char* a =
            reinterpret_cast<const __attribute__((address_space(3))) char*>((uintptr_t)(stage + (frag ^ ((uint32_t)sub << 5))));
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(a + O0));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(a + O1));
        return __builtin_bit_cast(i32x4_t, (v8s)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

__device__ __forceinline__ f32x4_t mfma_bf16(i32x4_t a, i32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// FA, FB: 0 e4m3, 1 e5m2.  Without scale operands (0) the instruction multiplies the plain values.
template <int FA, int FB>
__device__ __forceinline__ f32x4_t mfma_f8(i32x8_t a, i32x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, FA, FB, 0, 0, 0, 0);
}
__device__ __forceinline__ i32x8_t join(i32x4_t lo, i32x4_t hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// 8 8-bit values to bf16, which holds them exactly.  F: 0 e4m3, 1 e5m2.
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
template <int F>
__device__ __forceinline__ i32x4_t wide8(int lo, int hi) {
    auto two = [](int w, auto high) {
        if constexpr (F == 0)
            return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, high.value));
        else
            return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, high.value));
    };
    constexpr std::false_type l{};
    constexpr std::true_type h{};
    return i32x4_t{two(lo, l), two(lo, h), two(hi, l), two(hi, h)};
}

template <int F>
__device__ __forceinline__ void widen(i32x4_t lo, i32x4_t hi, i32x4_t (&w)[4]) {
    w[0] = wide8<F>(lo[0], lo[1]);
    w[1] = wide8<F>(lo[2], lo[3]);
    w[2] = wide8<F>(hi[0], hi[1]);
    w[3] = wide8<F>(hi[2], hi[3]);
}

// 4 neighbouring values of a row, the first n of them.
__device__ __forceinline__ void store4(uint64_t base, uint64_t i, uint32_t n, bool f32, f32x4_t v) {
    typedef f32x4_t f32x4_any __attribute__((aligned(4)));
    typedef u32x2_t u32x2_half __attribute__((aligned(2)));
    if (n >= 4) {
        if (f32)
            *at<f32x4_any>(base + i * 4) = v;
        else
            *at<u32x2_half>(base + i * 2) = u32x2_t{pack2(v[0], v[1]), pack2(v[2], v[3])};
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (e < n) {
                if (f32)
                    *at<float>(base, i + e) = v[e];
                else
                    *at<__bf16>(base, i + e) = (__bf16)v[e];
            }
    }
}
__device__ __forceinline__ f32x4_t load4(uint64_t base, uint64_t i, uint32_t n, bool f32) {
    typedef f32x4_t f32x4_any __attribute__((aligned(4)));
    typedef u32x2_t u32x2_half __attribute__((aligned(2)));
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n >= 4) {
        if (f32) return *at<const f32x4_any>(base + i * 4);
        const u32x2_t w = *at<const u32x2_half>(base + i * 2);
        return f32x4_t{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xFFFF0000u),
                       __builtin_bit_cast(float, w[1] << 16), __builtin_bit_cast(float, w[1] & 0xFFFF0000u)};
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (e < n) v[e] = f32 ? *at<const float>(base, i + e) : (float)*at<const __bf16>(base, i + e);
    return v;
}
__device__ __forceinline__ uint32_t left4(uint32_t n, uint32_t c) { return c < n ? min(n - c, 4u) : 0u; }

// ---- 8 bits ----------------------------------------------------------------------------
// C_mn = sum over blocks of K of sa[block][m] sb[block][n or its 128] (sum of the block's 128 products).
// The matrix unit sums a block from zero; the vector unit multiplies that by the scales and adds it to
// C in f32, 4 (one scale of B for a wave's columns) or 8 instructions for the 4 values of a matrix instruction.
//
// The 8-bit matrix instruction aligns the products of each 8 neighbouring values of K to the largest exponent
// among them and cuts what is below 2^-13 of that: 1e-5 to 7e-5 of the result (norm over norm; measured on normal
// values and on ones spread over 8 binades), far below bf16's own rounding but not below f32's.  So
// results in f32 (WIDE) come from bf16 matrix instructions, at half the rate, on the values converted in
// registers: their products and sums are exact to f32's rounding (6e-8 to 2e-7).
template <int BM, int BN, int WM, int WN, int NS, int FA, int FB, bool B_TILE, bool WIDE>
__device__ __forceinline__ void f8_tile(const T0gTileArgs& p) {
    constexpr int W = WM * WN, TM = BM / WM, TN = BN / WN, SM = TM / 16, SN = TN / 16;
    static_assert(!B_TILE || 128 % TN == 0, "one scale of B for a wave's columns");
    using OpA = RowsK<BM, W>;
    using OpB = RowsK<BN, W>;
    constexpr uint32_t A = OpA::kBytes, AB = A + OpB::kBytes, STAGE = AB + W * 256;
    static_assert(W * 64 == BM + BN || (W * 64 > BM + BN && W % 2 == 0), "a wave brings 64 scales");
    __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN, l16 = lane & 15u, q = lane >> 4;
    uint32_t tm, tn;
    tile_of(p, tm, tn);
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    OpA la;
    OpB lb;
    const uint32_t kb = (p.k + 15) & ~15u;   // whole pieces, zeros past k
    la.init(p.a, m0, p.m, p.lda, kb, wave, lane, wm * TM);
    lb.init(p.b, n0, p.n, p.ldb, kb, wave, lane, wn * TN);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    const uint32_t first = blockIdx.y * p.split_stages, end = min(first + p.split_stages, (p.k + 127) / 128);
    f32x4_t acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    // Scales, 64 a request: the first BM / 64 waves bring A's, the next BN / 64 B's.  A stage past the end brings zeros.
    const bool mine = wave < BM / 64;
    const uint32_t part = mine ? wave : wave - BM / 64;
    const uint32_t col = n0 + 64 * part + lane;   // with a scale for each 128 columns they are spread to the columns
    const uint64_t sbase = mine ? p.as : p.bs, sld = (uint64_t)(mine ? p.ldas : p.ldbs) * 4;
    const uint64_t sbytes = (uint64_t)(mine ? p.m : wave >= (BM + BN) / 64 ? 0u : B_TILE ? (p.n + 127) / 128 : p.n) * 4;
    const uint32_t soff = (mine ? m0 + 64 * part + lane : B_TILE ? col / 128 : col) * 4;
    auto issue = [&](uint32_t s, uint32_t lds) {
        la.issue(lds, s * 128, kb, wave);
        lb.issue(lds + A, s * 128, kb, wave);
        const u32x4_t r = rsrc_words_wide(sbase, (s < end ? sbytes : 0u) + s * sld, s * sld);
        dma4(r, soff, lds + AB + 256 * wave);
    };
    constexpr int kVmem = OpA::kInstr + OpB::kInstr + 1;
    for (int s = 0; s < NS - 1; ++s) issue(first + s, lds0 + s * STAGE);
    uint32_t cur = lds0, fill = lds0 + (NS - 1) * STAGE;
    for (uint32_t s = first; s < end; ++s) {
        // this stage is there (NS - 2 later ones may be on their way), and the one before is read
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        T0G_WAIT_VMCNT(kVmem * (NS - 2));
        barrier_no_fence();
        issue(s + NS - 1, fill);
        fill = fill + STAGE == lds0 + NS * STAGE ? lds0 : fill + STAGE;
        const uint32_t nxt = cur + STAGE == lds0 + NS * STAGE ? lds0 : cur + STAGE;
        f32x4_t sbv[B_TILE ? 1 : SN];
        float f[SM];
#pragma unroll
        for (int i = 0; i < SM; ++i) {
            f[i] = reinterpret_cast<const __attribute__((address_space(3))) float*>((uintptr_t)(cur + AB + (wm * TM + l16) * 4))[16 * i];
        }
        if constexpr (B_TILE) {
            const float sb = *reinterpret_cast<const __attribute__((address_space(3))) float*>((uintptr_t)(cur + AB + (BM + wn * TN) * 4));
#pragma unroll
            for (int i = 0; i < SM; ++i) f[i] *= sb;
        }
        if constexpr (!B_TILE)
#pragma unroll
            for (int j = 0; j < SN; ++j)
                sbv[j] = reinterpret_cast<const __attribute__((address_space(3))) f32x4_t*>(
                    (uintptr_t)(cur + AB + (BM + wn * TN + 4 * q) * 4))[4 * j];
        auto add = [&](int i, int j, int e, const f32x4_t& v) {
            acc[i][j][e] = __builtin_fmaf(B_TILE ? v[e] : v[e] * sbv[B_TILE ? 0 : j][e], f[i], acc[i][j][e]);
        };
        // The order of the instructions is pinned, the vector instructions on a result some matrix instructions
        // behind it: the compiler's own puts them right behind, where the wave waits for it.
        if constexpr (WIDE) {
            i32x4_t wb[SN][4], wa[2][4], lo = la.template read<0>(cur, 0), hi = la.template read<1>(cur, 0);
            f32x4_t v[2][SN];
#pragma unroll
            for (int j = 0; j < SN; ++j) widen<FB>(lb.template read<0>(cur + A, j), lb.template read<1>(cur + A, j), wb[j]);
            widen<FA>(lo, hi, wa[0]);
            // beside a row's 4 SN matrix instructions: the additions of the row before, and the conversion of the next
            static_assert(SN == 4, "16 additions of 4 values beside 16 matrix instructions");
#pragma unroll
            for (int i = 0; i < SM; ++i) {
                if (i + 1 < SM) {
                    lo = la.template read<0>(cur, i + 1);
                    hi = la.template read<1>(cur, i + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < 4 * SN; ++t) {
                    const int h = t / SN, j = t % SN;
                    v[i & 1][j] = mfma_bf16(wb[j][h], wa[i & 1][h], h ? v[i & 1][j] : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                    if (i > 0) add(i - 1, t / 4, t % 4, v[(i - 1) & 1][t / 4]);
                    if (i + 1 < SM && t >= 6 && t % 3 == 0) {
                        const int g = (t - 6) / 3;
                        wa[(i + 1) & 1][g] = g == 0   ? wide8<FA>(lo[0], lo[1])
                                             : g == 1 ? wide8<FA>(lo[2], lo[3])
                                             : g == 2 ? wide8<FA>(hi[0], hi[1])
                                                      : wide8<FA>(hi[2], hi[3]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int t = 0; t < 4 * SN; ++t) add(SM - 1, t / 4, t % 4, v[(SM - 1) & 1][t / 4]);
        } else {
            constexpr int kBehind = 3, T = SM * SN;
            i32x8_t fb[SN], fa[2];
            f32x4_t v[kBehind + 1];
            auto read_a = [&](int i) { fa[i & 1] = join(la.template read<0>(cur, i), la.template read<1>(cur, i)); };
            read_a(0);
#pragma unroll
            for (int j = 0; j < SN; ++j) fb[j] = join(lb.template read<0>(cur + A, j), lb.template read<1>(cur + A, j));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < T + kBehind; ++t) {
                if (t < T) {
                    v[t % (kBehind + 1)] = mfma_f8<FB, FA>(fb[t % SN], fa[t / SN & 1], f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
                    if (t % SN == 0 && t / SN + 1 < SM) read_a(t / SN + 1);
                }
                if (t >= kBehind)
#pragma unroll
                    for (int e = 0; e < 4; ++e) add((t - kBehind) / SN, (t - kBehind) % SN, e, v[(t - kBehind) % (kBehind + 1)]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        cur = nxt;
    }
    T0G_WAIT_VMCNT(0);   // stages past the end
    // a slice of K: f32 into its plane
    const uint64_t to = p.planes ? p.planes + (uint64_t)blockIdx.y * p.m * p.ldp * 4 : p.c;
    const uint32_t ld = p.planes ? p.ldp : p.ldc;
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        const uint32_t row = m0 + wm * TM + 16 * i + l16;
        if (row < p.m)
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                const uint32_t col = n0 + wn * TN + 16 * j + 4 * q;
                store4(to, (uint64_t)row * ld + col, left4(p.n, col), WIDE || p.planes, acc[i][j]);
            }
    }
}

// ---- gated -----------------------------------------------------------------------------
// g = x Wg^T and u = x Wu^T of the same columns in one wave: a tile has BN columns of each, and
// h = act(g) u is formed in registers.  GRAD: instead, with dh, dgate = dh u act'(g) and
// dup = dh act(g), from products that were not kept.
template <bool GRAD>
__device__ __forceinline__ void gated_out(const T0gTileArgs& p, uint32_t row, uint32_t col, f32x4_t g, f32x4_t u) {
    const uint32_t n = left4(p.n, col);
    f32x4_t a, d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float act, slope;
        activation(p.act, g[e], act, slope);
        a[e] = act;
        d[e] = slope;
    }
    if constexpr (GRAD) {
        const f32x4_t dh = load4(p.dh, (uint64_t)row * p.lddh + col, n, p.flags & T0G_TILE_DH_F32);
        store4(p.c, (uint64_t)row * p.ldc + col, n, false, dh * u * d);
        store4(p.c, (uint64_t)row * p.ldc + p.up_off + col, n, false, dh * a);
    } else {
        store4(p.c, (uint64_t)row * p.ldc + col, n, p.flags & T0G_TILE_OUT_F32, a * u);
        if (p.gate) store4(p.gate, (uint64_t)row * p.ldg + col, n, false, g);
        if (p.up) store4(p.up, (uint64_t)row * p.ldg + col, n, false, u);
    }
}

template <int BM, int BN, int WM, int WN, int NS, bool NC, bool GRAD>
__device__ __forceinline__ void gated_tile(const T0gTileArgs& p) {
    constexpr int W = WM * WN, TM = BM / WM, TN = BN / WN, SM = TM / 16, SN = TN / 16;
    using OpA = RowsK<BM, W>;
    using OpB = typename std::conditional<NC, RowsN<BN, W>, RowsK<BN, W>>::type;
    constexpr uint32_t A = OpA::kBytes, B = OpB::kBytes, STAGE = A + 2 * B;
    __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN, l16 = lane & 15u, q = lane >> 4;
    uint32_t tm, tn;
    tile_of(p, tm, tn);
    const uint32_t m0 = tm * BM, n0 = tn * BN;
    OpA la;
    OpB lg, lu;
    const uint32_t kb = (p.k * 2 + 15) & ~15u;
    la.init(p.a, m0, p.m, (uint64_t)p.lda * 2, kb, wave, lane, wm * TM);
    if constexpr (NC) {
        lg.init(p.b, n0, p.n, p.k, p.ldb, wave, lane, wn * TN);
        lu.init(p.b2, n0, p.n, p.k, p.ldb, wave, lane, wn * TN);
    } else {
        lg.init(p.b, n0, p.n, (uint64_t)p.ldb * 2, kb, wave, lane, wn * TN);
        lu.init(p.b2, n0, p.n, (uint64_t)p.ldb * 2, kb, wave, lane, wn * TN);
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    const uint32_t first = blockIdx.y * p.split_stages, end = min(first + p.split_stages, (p.k + 63) / 64);
    f32x4_t g[SM][SN], u[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; ++i)
#pragma unroll
        for (int j = 0; j < SN; ++j) g[i][j] = u[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    auto issue = [&](uint32_t s, uint32_t lds) {   // past the end: zeros
        la.issue(lds, s * 128, kb, wave);
        if constexpr (NC) {
            lg.issue(lds + A, s * 64, p.k, wave, lane);
            lu.issue(lds + A + B, s * 64, p.k, wave, lane);
        } else {
            lg.issue(lds + A, s * 128, kb, wave);
            lu.issue(lds + A + B, s * 128, kb, wave);
        }
    };
    constexpr int kVmem = OpA::kInstr + 2 * OpB::kInstr;
    for (int s = 0; s < NS - 1; ++s) issue(first + s, lds0 + s * STAGE);
    uint32_t cur = lds0, fill = lds0 + (NS - 1) * STAGE;
    for (uint32_t s = first; s < end; ++s) {
        // this stage is there (NS - 2 later ones may be on their way), and the one before is read
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        T0G_WAIT_VMCNT(kVmem * (NS - 2));
        barrier_no_fence();
        issue(s + NS - 1, fill);
        fill = fill + STAGE == lds0 + NS * STAGE ? lds0 : fill + STAGE;
        const uint32_t nxt = cur + STAGE == lds0 + NS * STAGE ? lds0 : cur + STAGE;
        auto half = [&](auto h) {
            constexpr int H = h.value;
            i32x4_t fg[SN], fu[SN];
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                fg[j] = lg.template read<H>(cur + A, j);
                fu[j] = lu.template read<H>(cur + A + B, j);
            }
#pragma unroll
            for (int i = 0; i < SM; ++i) {
                const i32x4_t fa = la.template read<H>(cur, i);
#pragma unroll
                for (int j = 0; j < SN; ++j) {
                    g[i][j] = mfma_bf16(fg[j], fa, g[i][j]);
                    u[i][j] = mfma_bf16(fu[j], fa, u[i][j]);
                }
            }
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
        cur = nxt;
    }
    T0G_WAIT_VMCNT(0);   // stages past the end
#pragma unroll
    for (int i = 0; i < SM; ++i) {
        const uint32_t row = m0 + wm * TM + 16 * i + l16;
        if (row < p.m)
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                const uint32_t col = n0 + wn * TN + 16 * j + 4 * q;
                if (p.planes) {   // a slice of K
                    const uint64_t to = p.planes + 2 * (uint64_t)blockIdx.y * p.m * p.ldp * 4;
                    store4(to, (uint64_t)row * p.ldp + col, left4(p.n, col), true, g[i][j]);
                    store4(to + (uint64_t)p.m * p.ldp * 4, (uint64_t)row * p.ldp + col, left4(p.n, col), true, u[i][j]);
                } else {
                    gated_out<GRAD>(p, row, col, g[i][j], u[i][j]);
                }
            }
    }
}

// The slices of K in their order, 4 columns a thread.
__device__ __forceinline__ void join_slices(const T0gJoinArgs& a) {
    const T0gTileArgs& p = a.t;
    const uint32_t per_row = p.ldp / 4;
    const uint64_t plane = (uint64_t)p.m * p.ldp * 4;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < p.m * per_row; i += gridDim.x * 256) {   // below 2^31: the host's
        const uint32_t row = i / per_row, col = 4 * (i - row * per_row);
        const uint64_t at_ = p.planes + (uint64_t)i * 16;
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f}, u = v;
        if (col >= p.n) continue;
        for (uint32_t s = 0; s < a.slices; ++s) {
            if (a.gated) {
                v += *at<const f32x4_t>(at_ + 2 * s * plane);
                u += *at<const f32x4_t>(at_ + (2 * s + 1) * plane);
            } else {
                v += *at<const f32x4_t>(at_ + s * plane);
            }
        }
        if (a.gated == 2)
            gated_out<true>(p, row, col, v, u);
        else if (a.gated)
            gated_out<false>(p, row, col, v, u);
        else
            store4(p.c, (uint64_t)row * p.ldc + col, left4(p.n, col), p.flags & T0G_TILE_OUT_F32, v);
    }
}

}  // namespace t0g

#endif
