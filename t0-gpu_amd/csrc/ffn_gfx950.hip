// Operators of a model's feed-forward layer for MI355X (gfx950): its norm, values in 8 bits with
// block scales, their product, and the gated pair of projections with its gradient.
#define T0G_TILES_ONLY
#include "gemm_gfx950.hip"
#include "ffn_rows.h"
#include "ffn_tile.h"
#include "ffn_skinny.h"
#include "ffn_big.h"
#include "ffn_gated.h"

// Symbols: t0g_ffn_norm[_grad]_<threads of a row>x<pieces of a thread>[_fast].
#define NORM(NT, CH, R, SUFFIX, FAST)                                                                      \
    extern "C" __global__ void __launch_bounds__(NT * R) t0g_ffn_norm_##NT##x##CH##SUFFIX(T0gNormArgs p) { \
        t0g::rms_norm<NT, CH, R, FAST>(p);                                                                 \
    }
NORM(64, 1, 4, , false)
NORM(256, 1, 1, , false)
NORM(256, 2, 1, , false)
NORM(512, 2, 1, , false)
NORM(1024, 2, 1, , false)
NORM(64, 1, 4, _fast, true)
NORM(256, 1, 1, _fast, true)
NORM(256, 2, 1, _fast, true)
NORM(512, 2, 1, _fast, true)
NORM(1024, 2, 1, _fast, true)
#define NORM_GRAD(NT, CH, R, SUFFIX, FAST, KEEP, PRE)                                                              \
    extern "C" __global__ void __launch_bounds__(NT * R) t0g_ffn_norm_grad_##NT##x##CH##SUFFIX(T0gNormGradArgs p) { \
        t0g::rms_norm_grad<NT, CH, R, FAST, KEEP, PRE>(p);                                                         \
    }
NORM_GRAD(64, 1, 4, , false, true, false)
NORM_GRAD(256, 1, 1, , false, true, false)
NORM_GRAD(256, 2, 1, , false, true, false)
NORM_GRAD(512, 2, 1, , false, true, false)
NORM_GRAD(1024, 2, 1, , false, false, false)
NORM_GRAD(64, 1, 4, _fast, true, true, true)
NORM_GRAD(256, 1, 1, _fast, true, true, true)
NORM_GRAD(256, 2, 1, _fast, true, true, true)
NORM_GRAD(512, 2, 1, _fast, true, true, true)
NORM_GRAD(1024, 2, 1, _fast, true, true, false)
extern "C" __global__ void __launch_bounds__(1024) t0g_ffn_column_sum(T0gColSumArgs p) { t0g::column_sum(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_quantize_rows(T0gQuantArgs p) { t0g::quantize_rows<false>(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_quantize_rows_fast(T0gQuantArgs p) { t0g::quantize_rows<true>(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_quantize_tile(T0gQuantArgs p) { t0g::quantize_tile<false>(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_quantize_tile_fast(T0gQuantArgs p) { t0g::quantize_tile<true>(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_gated_grad(T0gGatedGradArgs p) { t0g::gated_grad(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_pad_rows(T0gPadArgs p) { t0g::pad_rows(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_join_slices(T0gJoinArgs p) { t0g::join_slices(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_ffn_add_planes(T0gAddArgs p) { t0g::add_planes(p); }

// Symbols: t0g_ffn_f8_<tile>_<type of A><type of B>_<blocks of B>_<output type>.
#define F8_KERNEL(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB, BLOCK, B_TILE, OUT, WIDE)                                                   \
    extern "C" __global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2)))                     \
        t0g_ffn_f8_##NAME##_##TYPES##_##BLOCK##_##OUT(T0gTileArgs p) {                                                        \
        t0g::f8_tile<BM, BN, WM, WN, NS, FA, FB, B_TILE, WIDE>(p);                                                               \
    }
#define F8_TYPES(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB)                        \
    F8_KERNEL(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB, tile, true, bf16, false)  \
    F8_KERNEL(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB, tile, true, f32, true)    \
    F8_KERNEL(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB, row, false, bf16, false)  \
    F8_KERNEL(NAME, BM, BN, WM, WN, NS, TYPES, FA, FB, row, false, f32, true)
#define F8_TILES(NAME, BM, BN, WM, WN, NS)             \
    F8_TYPES(NAME, BM, BN, WM, WN, NS, e4e4, 0, 0)     \
    F8_TYPES(NAME, BM, BN, WM, WN, NS, e4e5, 0, 1)     \
    F8_TYPES(NAME, BM, BN, WM, WN, NS, e5e4, 1, 0)     \
    F8_TYPES(NAME, BM, BN, WM, WN, NS, e5e5, 1, 1)
F8_TILES(128x128, 128, 128, 2, 2, 2)
F8_TILES(64x128, 64, 128, 2, 2, 3)

#define F8_BIG(TYPES, FA, FB)                                                                                   \
    extern "C" __global__ void __launch_bounds__(512) t0g_ffn_f8_256x256_##TYPES##_tile_bf16(T0gTileArgs p) {   \
        t0g::f8_big<FA, FB, true>(p);                                                                           \
    }                                                                                                           \
    extern "C" __global__ void __launch_bounds__(512) t0g_ffn_f8_256x256_##TYPES##_row_bf16(T0gTileArgs p) {    \
        t0g::f8_big<FA, FB, false>(p);                                                                          \
    }
F8_BIG(e4e4, 0, 0)
F8_BIG(e4e5, 0, 1)
F8_BIG(e5e4, 1, 0)
F8_BIG(e5e5, 1, 1)
#define F8_SKINNY(MT, TYPES, FA, FB)                                                                              \
    extern "C" __global__ void __launch_bounds__(512) t0g_ffn_f8_skinny##MT##_##TYPES##_tile(T0gTileArgs p) {      \
        t0g::f8_skinny<8, MT, FA, FB, true>(p);                                                                    \
    }                                                                                                              \
    extern "C" __global__ void __launch_bounds__(512) t0g_ffn_f8_skinny##MT##_##TYPES##_row(T0gTileArgs p) {       \
        t0g::f8_skinny<8, MT, FA, FB, false>(p);                                                                   \
    }
#define F8_SKINNIES(MT)          \
    F8_SKINNY(MT, e4e4, 0, 0)    \
    F8_SKINNY(MT, e4e5, 0, 1)    \
    F8_SKINNY(MT, e5e4, 1, 0)    \
    F8_SKINNY(MT, e5e5, 1, 1)
F8_SKINNIES(1)
F8_SKINNIES(2)
extern "C" __global__ void __launch_bounds__(512) t0g_ffn_gated_skinny1(T0gTileArgs p) { t0g::gated_skinny<8, 1>(p); }
extern "C" __global__ void __launch_bounds__(512) t0g_ffn_gated_skinny2(T0gTileArgs p) { t0g::gated_skinny<8, 2>(p); }

#define GATED(NAME, BM, BN, WM, WN, NS)                                                                            \
    extern "C" __global__ void __launch_bounds__(64 * WM * WN) t0g_ffn_gated_##NAME##_nt(T0gTileArgs p) {      \
        t0g::gated_tile<BM, BN, WM, WN, NS, false, false>(p);                                                      \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(64 * WM * WN) t0g_ffn_gated_##NAME##_nn(T0gTileArgs p) {      \
        t0g::gated_tile<BM, BN, WM, WN, NS, true, false>(p);                                                       \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(64 * WM * WN) t0g_ffn_gated_##NAME##_nt_grad(T0gTileArgs p) { \
        t0g::gated_tile<BM, BN, WM, WN, NS, false, true>(p);                                                       \
    }                                                                                                          \
    extern "C" __global__ void __launch_bounds__(64 * WM * WN) t0g_ffn_gated_##NAME##_nn_grad(T0gTileArgs p) { \
        t0g::gated_tile<BM, BN, WM, WN, NS, true, true>(p);                                                        \
    }
GATED(128x64, 128, 64, 2, 2, 2)
GATED(64x64, 64, 64, 2, 2, 3)
extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) t0g_ffn_gated_256x128_nt(T0gTileArgs p) {
    t0g::gated_big<false>(p);
}
extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) t0g_ffn_gated_256x128_nn(T0gTileArgs p) {
    t0g::gated_big<true>(p);
}
