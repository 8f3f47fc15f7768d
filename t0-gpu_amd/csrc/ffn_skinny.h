// Products of few rows (up to 32): C = A B^T is bound by reading B once, so no operand goes through LDS.
// A workgroup takes 16 columns of C (gated: 16 of each product); its waves take the 128-byte
// blocks of K in turn, so together they read a contiguous piece of each of the 16 rows of B, and add
// up through LDS in the order of the waves.  A lane's share of a block is two 16-byte pieces at the places where
// the matrix unit wants them; rows may start at any element.
#ifndef T0G_FFN_SKINNY_H
#define T0G_FFN_SKINNY_H

namespace t0g {

typedef i32x4_t i32x4_any __attribute__((aligned(1)));

// Bytes [at, at + 16) of a row that ends at `end`, zeros past it.
__device__ __forceinline__ i32x4_t load16(uint64_t row, uint32_t at_, uint32_t end) {
    if (at_ + 16 <= end) return *at<const i32x4_any>(row + at_);
    return at_ < end ? __builtin_bit_cast(i32x4_t, tail16(row, at_, end)) : i32x4_t{0, 0, 0, 0};
}

template <int ROWS16>
struct Pieces {
    i32x4_t lo[ROWS16], hi[ROWS16];
    // Block `blk` of 16 ROWS16 rows from `base`; lane (q, l16): chunks q and 4 + q of row l16 of each 16.
    __device__ __forceinline__ void load(const uint64_t (&row)[ROWS16], uint32_t blk, uint32_t q, uint32_t bytes, bool tail) {
        const uint32_t a = blk * 128 + 16 * q;
#pragma unroll
        for (int i = 0; i < ROWS16; ++i) {
            if (tail) {
                lo[i] = load16(row[i], a, bytes);
                hi[i] = load16(row[i], a + 64, bytes);
            } else {
                lo[i] = *at<const i32x4_any>(row[i] + a);
                hi[i] = *at<const i32x4_any>(row[i] + a + 64);
            }
        }
    }
};

// The waves' sums v[T] (T sub-tiles of 16 x 16), added up in their order; true in the waves t < T that then hold
// sub-tile t in v[0].
template <int W, int T>
__device__ __forceinline__ bool add_waves(f32x4_t (&v)[T], f32x4_t (*lds)[T][64], uint32_t wave, uint32_t lane) {
#pragma unroll
    for (int t = 0; t < T; ++t) lds[wave][t][lane] = v[t];
    __syncthreads();
    if (wave >= T) return false;
    f32x4_t s = lds[0][wave][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += lds[w][wave][lane];
    v[0] = s;
    return true;
}

// U blocks of a wave are in flight at once.
template <int W, int MT, int FA, int FB, bool B_TILE>
__device__ __forceinline__ void f8_skinny(const T0gTileArgs& p) {
    constexpr int U = MT == 1 ? 4 : 2;
    __shared__ f32x4_t sums[W][MT][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t l16 = lane & 15u, q = lane >> 4, n0 = 16 * blockIdx.x;
    const uint64_t brow[1] = {p.b + (uint64_t)min(n0 + l16, p.n - 1) * p.ldb};   // rows past the end: the last again, not stored
    uint64_t arow[MT];
    uint32_t m[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] = min(16 * t + l16, p.m - 1);
        arow[t] = p.a + (uint64_t)m[t] * p.lda;
    }
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t blocks = (p.k + 127) / 128, full = p.k / 128;
    Pieces<1> b[U];
    Pieces<MT> a[U];
    float sa[U][MT];
    f32x4_t sb[U];
    auto load = [&](int u, uint32_t blk, bool tail) {
        b[u].load(brow, blk, q, p.k, tail);
        a[u].load(arow, blk, q, p.k, tail);
#pragma unroll
        for (int t = 0; t < MT; ++t) sa[u][t] = *at<const float>(p.as, (uint64_t)blk * p.ldas + m[t]);
        if constexpr (B_TILE) {
            const float s = *at<const float>(p.bs, (uint64_t)blk * p.ldbs + n0 / 128);
            sb[u] = f32x4_t{s, s, s, s};
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) sb[u][e] = *at<const float>(p.bs, (uint64_t)blk * p.ldbs + min(n0 + 4 * q + e, p.n - 1));
        }
    };
    auto multiply = [&](int u) {
        i32x4_t wb[4];
        widen<FB>(b[u].lo[0], b[u].hi[0], wb);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            i32x4_t wa[4];
            widen<FA>(a[u].lo[t], a[u].hi[t], wa);
            f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 4; ++h) v = mfma_bf16(wb[h], wa[h], v);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(v[e] * sb[u][e], sa[u][t], acc[t][e]);
        }
    };
    uint32_t blk = wave;
    for (; blk + (U - 1) * W < full; blk += U * W) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(u, blk + u * W, false);
        __builtin_amdgcn_sched_barrier(0);   // all of them on their way before the first is waited for
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(u);
    }
    for (; blk < blocks; blk += W) {
        load(0, blk, blk >= full);
        multiply(0);
    }
    if (add_waves<W, MT>(acc, sums, wave, lane)) {
        const uint32_t row = 16 * wave + l16, col = n0 + 4 * q;
        if (row < p.m) store4(p.c, (uint64_t)row * p.ldc + col, left4(p.n, col), p.flags & T0G_TILE_OUT_F32, acc[0]);
    }
}

template <int W, int MT>
__device__ __forceinline__ void gated_skinny(const T0gTileArgs& p) {
    constexpr int U = MT == 1 ? 4 : 2;
    __shared__ f32x4_t sums[W][2 * MT][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t l16 = lane & 15u, q = lane >> 4, n0 = 16 * blockIdx.x, kb = p.k * 2;
    const uint64_t wrow = (uint64_t)min(n0 + l16, p.n - 1) * p.ldb * 2;
    const uint64_t brow[2] = {p.b + wrow, p.b2 + wrow};
    uint64_t arow[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) arow[t] = p.a + (uint64_t)min(16 * t + l16, p.m - 1) * p.lda * 2;
    f32x4_t acc[2 * MT];   // both products of each 16 rows
#pragma unroll
    for (int t = 0; t < 2 * MT; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t blocks = (kb + 127) / 128, full = kb / 128;
    Pieces<2> b[U];
    Pieces<MT> a[U];
    auto load = [&](int u, uint32_t blk, bool tail) {
        b[u].load(brow, blk, q, kb, tail);
        a[u].load(arow, blk, q, kb, tail);
    };
    auto multiply = [&](int u) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                acc[2 * t + s] = mfma_bf16(b[u].lo[s], a[u].lo[t], acc[2 * t + s]);
                acc[2 * t + s] = mfma_bf16(b[u].hi[s], a[u].hi[t], acc[2 * t + s]);
            }
    };
    uint32_t blk = wave;
    for (; blk + (U - 1) * W < full; blk += U * W) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(u, blk + u * W, false);
        __builtin_amdgcn_sched_barrier(0);   // all of them on their way before the first is waited for
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(u);
    }
    for (; blk < blocks; blk += W) {
        load(0, blk, blk >= full);
        multiply(0);
    }
    // the waves' sums in their order; wave t then holds both products of rows 16 t .. + 15
#pragma unroll
    for (int t = 0; t < 2 * MT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave >= MT) return;
    f32x4_t g = sums[0][2 * wave][lane], u = sums[0][2 * wave + 1][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) {
        g += sums[w][2 * wave][lane];
        u += sums[w][2 * wave + 1][lane];
    }
    const uint32_t row = 16 * wave + l16, col = n0 + 4 * q;
    if (row < p.m) gated_out<false>(p, row, col, g, u);
}

}  // namespace t0g

#endif
