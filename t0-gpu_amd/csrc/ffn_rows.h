// Row kernels of the feed-forward layer's operators: root-mean-square norms and their
// gradients, values in 8 bits with block scales, and the element-wise passes around the
// products.  All of them read and write memory once and are bound by it.  A lane takes 8
// neighbouring values of a row (16 bytes of bf16), so 16 lanes, a DPP row, take the 128 that
// share a scale.  Rows may start at any element: vector accesses need no alignment here, and
// a row's last piece, if it is not whole, goes value by value.
#ifndef T0G_FFN_ROWS_H
#define T0G_FFN_ROWS_H

namespace t0g {

typedef u32x4_t u32x4_any __attribute__((aligned(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any __attribute__((aligned(1)));
typedef u32x4_t u32x4_byte __attribute__((aligned(1)));
template <class T>
using gptr = __attribute__((address_space(1))) T*;
template <class T>
__device__ __forceinline__ gptr<T> at(uint64_t base, uint64_t i = 0) {
    return reinterpret_cast<gptr<T>>((uintptr_t)base) + i;
}

// ---- lanes -----------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_row(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// NaN passes on: a block that holds one has a NaN for its scale.
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
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row16_sum(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// N sums over the workgroup's W waves; `t`: N W floats of LDS, not in use by the reduction before.
template <int W, int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* t) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63u) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) t[i * W + (threadIdx.x >> 6)] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = t[i * W];
#pragma unroll
            for (int w = 1; w < W; ++w) v[i] += t[i * W + w];
        }
    }
}

// ---- 8 values of a row -----------------------------------------------------------------
struct Raw8 {
    u32x4_t lo, hi;   // 8 bf16 in lo, or 8 f32
};
// The values [i, i + n) at base, n <= 8; zeros for the rest.
__device__ __forceinline__ Raw8 load8(uint64_t base, uint64_t i, uint32_t n, bool f32) {
    Raw8 r = {u32x4_t{0u, 0u, 0u, 0u}, u32x4_t{0u, 0u, 0u, 0u}};
    if (n >= 8) {
        if (f32) {
            const gptr<const u32x4_any> p = at<const u32x4_any>(base + i * 4);
            r.lo = p[0];
            r.hi = p[1];
        } else {
            r.lo = *at<const u32x4_any>(base + i * 2);
        }
    } else if (n > 0) {
        if (f32) {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (e < n) (e < 4 ? r.lo : r.hi)[e & 3] = *at<const uint32_t>(base, i + e);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (e < n) r.lo[e / 2] |= (uint32_t)*at<const uint16_t>(base, i + e) << (16 * (e & 1));
        }
    }
    return r;
}
__device__ __forceinline__ void values8(const Raw8& r, bool f32, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t w = f32 ? (e < 4 ? r.lo[e] : r.hi[e - 4]) : (e & 1 ? r.lo[e / 2] & 0xFFFF0000u : r.lo[e / 2] << 16);
        v[e] = __builtin_bit_cast(float, w);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
}
__device__ __forceinline__ void store8(uint64_t base, uint64_t i, uint32_t n, bool f32, const float (&v)[8]) {
    if (n >= 8) {
        if (f32) {
            const gptr<u32x4_any> p = at<u32x4_any>(base + i * 4);
            p[0] = __builtin_bit_cast(u32x4_t, f32x4_t{v[0], v[1], v[2], v[3]});
            p[1] = __builtin_bit_cast(u32x4_t, f32x4_t{v[4], v[5], v[6], v[7]});
        } else {
            *at<u32x4_any>(base + i * 2) = u32x4_t{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            if (e < n) {
                if (f32)
                    *at<float>(base, i + e) = v[e];
                else
                    *at<__bf16>(base, i + e) = (__bf16)v[e];
            }
    }
}

// ---- 8 bits ----------------------------------------------------------------------------
// A block's scale is max(largest magnitude, 2^-100) / the type's largest value: 0.5 units of
// its 4 or 3 bits is then all that a value loses, and a block of zeros has a scale too.
// A value is multiplied by the quotient's inverse in two parts, inv + rest, which is within 2^-45 of it, and the
// product rounded once to f32.  Quotients on a border between two roundings are common among bf16 values: with the
// inverse in one part 3e-4 of normal values went to the wrong side.  Such a quotient has few bits, so that
// it comes out as it is and goes to the even neighbour; the others of bf16 values are 2^-14 of themselves away
// from a border or more.  With a NaN or an infinity among them all of a block's values come out as NaN.
constexpr float kLeastAmax = 7.888609052210118e-31f;   // 2^-100
__device__ __forceinline__ float f8_most(bool e5m2) { return e5m2 ? 57344.0f : 448.0f; }
struct BlockScale {
    float scale, inv, rest;
};
// `factor`: what all of the block's values (and amax) are yet to be multiplied by.  It is no part of the quotients,
// which so have no rounding of it, but where the least scale takes over.
__device__ __forceinline__ BlockScale block_scale(float amax, bool e5m2, float factor = 1.0f) {
    const float most = f8_most(e5m2), top = amax * factor;
    amax = top < kLeastAmax ? kLeastAmax / factor : amax;
    float inv = most / amax, r = __builtin_fmaf(-inv, amax, most);
    // rounded down, so that rest is not negative and zeros keep their sign
    inv = r < 0.0f ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, inv) - 1u) : inv;
    r = __builtin_fmaf(-inv, amax, most);
    return BlockScale{max_(top, kLeastAmax) / most, inv, r > 0.0f ? r * (e5m2 ? 1.0f / 57344.0f : 1.0f / 448.0f) * inv : 0.0f};
}
__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = __builtin_fabsf(v[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) m = max_(m, __builtin_fabsf(v[e]));
    return m;
}
__device__ __forceinline__ uint32_t f8x4(float a, float b, float c, float d, bool e5m2) {
    int w = 0;
    if (e5m2) {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
    return (uint32_t)w;
}
__device__ __forceinline__ u32x2_t f8x8(const float (&v)[8], float inv, float rest, bool e5m2) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = __builtin_fmaf(v[e], inv, v[e] * rest);
    return u32x2_t{f8x4(t[0], t[1], t[2], t[3], e5m2), f8x4(t[4], t[5], t[6], t[7], e5m2)};
}
__device__ __forceinline__ void store_f8x8(uint64_t addr, uint32_t n, u32x2_t w) {
    if (n >= 8) {
        *at<u32x2_any>(addr) = w;
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            if (e < n) *at<uint8_t>(addr, e) = (uint8_t)(w[e / 4] >> (8 * (e & 3)));
    }
}

// Valid values of the piece of 8 at column c of a row of `cols`; FAST: of whole pieces.
template <bool FAST = false>
__device__ __forceinline__ uint32_t left8(uint32_t cols, uint32_t c) {
    return c < cols ? (FAST ? 8u : min(cols - c, 8u)) : 0u;
}

// n as a new value to the compiler, which otherwise forms the lane masks of all comparisons with it before the
// loop over the rows and runs out of scalar registers.
template <bool DO>
__device__ __forceinline__ uint32_t anew(uint32_t n) {
    if constexpr (DO) asm volatile("" : "+v"(n));
    return n;
}

// ---- the norm --------------------------------------------------------------------------
// What a row's values are multiplied by: 1, or a power of two where f32 does not hold the sum of their squares (16384
// of values up to 2^128, or squares that it would lose and that count, with so small an eps).  They are then
// added up again, and rho is theirs: s rho stays the same, and rho^2 and 1 / rho^2 are always f32's.  The same in all
// threads of the row.
__device__ __forceinline__ float range_scale(float sum, float eps) {
    const float k = sum > 0x1p96f ? 0x1p-80f : sum < 0x1p-90f && eps < 0x1p-60f ? 0x1p90f : 1.0f;
    return __builtin_bit_cast(float, uniform_u32(__builtin_bit_cast(uint32_t, k)));
}
// y = s rho (w + offset), rho = (mean s^2 + eps)^-1/2, s = x + residual.  NT threads take a row, with CH pieces
// of 8 each, and keep it in registers between the sum of squares and the output: memory is read and
// written once.  Rows of one wave go R to a workgroup.  FAST: bf16 inputs of whole pieces of 8, which need
// half the registers: 8192x4096 with the residual into e4m3 in 44 us that way, 53 with types and ends
// looked at in the kernel.
template <int NT, int CH, int R, bool FAST>
__device__ __forceinline__ void rms_norm(const T0gNormArgs& p) {
    constexpr int W = NT / 64;
    static_assert(R == 1 || NT == 64, "several rows: a wave each");
    __shared__ float t[2][W];
    const bool xf = !FAST && p.flags & T0G_ROWS_X_F32, rf = !FAST && p.flags & T0G_ROWS_R_F32, wf = !FAST && p.flags & T0G_ROWS_W_F32,
               e5m2 = p.flags & T0G_ROWS_E5M2;
    const uint32_t first = threadIdx.x % NT, step = gridDim.x * R;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x * R + threadIdx.x / NT; row < p.rows; row += step, turn ^= 1) {
        Raw8 x[CH], r[CH], w[CH];
        auto load = [&](int i) {
            const uint32_t c = 8 * (i * NT + first), n = anew<!FAST && (CH > 1)>(left8<FAST>(p.hidden, c));
            x[i] = load8(p.x, (uint64_t)row * p.ldx + c, n, xf);
            if (p.residual) r[i] = load8(p.residual, (uint64_t)row * p.ldr + c, n, rf);
            if (p.weight) w[i] = load8(p.weight, c, n, wf);
        };
#pragma unroll
        for (int i = 0; i < CH; ++i) load(i);
        float s[CH][8], sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            values8(x[i], xf, s[i]);
            if (p.residual) {
                float d[8];
                values8(r[i], rf, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[i][e] += d[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[0] = __builtin_fmaf(s[i][e], s[i][e], sum[0]);
        }
        if (p.sum)
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint32_t c = 8 * (i * NT + first);
                store8(p.sum, (uint64_t)row * p.ldsum + c, anew<!FAST && (CH > 1)>(left8<FAST>(p.hidden, c)), p.flags & T0G_ROWS_OUT_F32, s[i]);
            }
        block_sum<W>(sum, t[turn]);
        float eps = p.eps;
        const float k = range_scale(sum[0], eps);
        if (k != 1.0f) {
            sum[0] = 0.0f;
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    s[i][e] *= k;
                    sum[0] = __builtin_fmaf(s[i][e], s[i][e], sum[0]);
                }
            eps = eps * k * k;
            turn ^= 1;
            block_sum<W>(sum, t[turn]);
        }
        const float rho = 1.0f / __builtin_sqrtf(sum[0] / (float)p.hidden + eps);
        // as a power of two, which rounds nothing and keeps s (w + offset) in range, times a value from 1 to 2
        const uint32_t bits = __builtin_bit_cast(uint32_t, rho);
        const float rho2 = __builtin_bit_cast(float, bits & 0x7F800000u);
        const float rest = rho == rho ? __builtin_bit_cast(float, (bits & 0x007FFFFFu) | 0x3F800000u) : rho;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = 8 * (i * NT + first), n = anew<!FAST && (CH > 1)>(left8<FAST>(p.hidden, c));
            float v[8], g[8];
            if (p.weight) {
                values8(w[i], wf, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] += p.weight_offset;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = 1.0f;
            }
            if (p.y) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = s[i][e] * rho * g[e];
                store8(p.y, (uint64_t)row * p.ldy + c, n, p.flags & T0G_ROWS_Y_F32, v);
            }
            if (p.q) {
                // a row's last piece holds zeros past its values, for any rho but an infinite one
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] = e < n ? s[i][e] * rho2 * g[e] : 0.0f;
                const BlockScale b = block_scale(row16_max(amax8(v)), e5m2, rest);
                store_f8x8(p.q + (uint64_t)row * p.ldq + c, n, f8x8(v, b.inv, b.rest, e5m2));
                if ((threadIdx.x & 15u) == 0 && n) *at<float>(p.scales, (uint64_t)(c / T0G_SCALE_BLOCK) * p.ldsc + row) = b.scale;
            }
        }
    }
}

// With n = s rho and g = dy (w + offset):  ds = rho (g - n mean(g n)) + dsum,  dw = sum over rows of dy n.
// mean(g n) = rho mean(g s), so one pass over the row gives both sums.  NT threads take a row, R rows a workgroup,
// which goes on to every gridDim.x-th of them.  Each thread adds up its part of dw in registers, in the order of
// its rows.  FAST: bf16 inputs of whole pieces of 8.  PRE: the next row's are on their way while this one's
// sums are formed.  KEEP: the row stays in registers between the sums and ds; else it is read again, from the caches.
template <int NT, int CH, int R, bool FAST, bool KEEP, bool PRE>
__device__ __forceinline__ void rms_norm_grad(const T0gNormGradArgs& p) {
    constexpr int W = NT / 64;
    static_assert(R == 1 || (NT == 64 && CH == 1), "several rows: a wave each");
    __shared__ float t[2][2 * W];
    const bool yf = !FAST && p.flags & T0G_ROWS_Y_F32, xf = !FAST && p.flags & T0G_ROWS_X_F32, wf = !FAST && p.flags & T0G_ROWS_W_F32,
               sf = !FAST && p.flags & T0G_ROWS_R_F32;
    const uint32_t first = threadIdx.x % NT;
    float dw[CH][8];
    Raw8 w[KEEP ? CH : 1];
    auto load_weight = [&](int i) {
        const uint32_t c = 8 * (i * NT + first);
        if (p.weight) w[KEEP ? i : 0] = load8(p.weight, c, anew<!FAST && (CH > 1)>(left8<FAST>(p.hidden, c)), wf);
    };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if constexpr (KEEP) load_weight(i);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
    }
    auto weight = [&](int i, float (&v)[8]) {
        if (p.weight) {
            values8(w[KEEP ? i : 0], wf, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += p.weight_offset;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 1.0f;
        }
    };
    constexpr int K = KEEP ? CH : 1;
    Raw8 y[K], x[K], d[K];
    auto load = [&](uint32_t row, int i, Raw8& yi, Raw8& xi, Raw8& di) {
        const uint32_t c = 8 * (i * NT + first), n = anew<!FAST && (CH > 1)>(row < p.rows ? left8<FAST>(p.hidden, c) : 0u);
        yi = load8(p.dy, (uint64_t)row * p.lddy + c, n, yf);
        xi = load8(p.x, (uint64_t)row * p.ldx + c, n, xf);
        if (p.dsum && p.dx) di = load8(p.dsum, (uint64_t)row * p.ldds + c, n, sf);
    };
    uint32_t turn = 0, row = blockIdx.x * R + threadIdx.x / NT;
    const uint32_t step = gridDim.x * R;
    if constexpr (PRE)
#pragma unroll
        for (int i = 0; i < CH; ++i) load(row, i, y[i], x[i], d[i]);
    for (; row < p.rows; row += step, turn ^= 1) {
        Raw8 y2[K], x2[K], d2[K];
        if constexpr (PRE)   // row + step below 2^32: both are below 2^31
#pragma unroll
            for (int i = 0; i < CH; ++i) load(row + step, i, y2[i], x2[i], d2[i]);
        else if constexpr (KEEP)
#pragma unroll
            for (int i = 0; i < CH; ++i) load(row, i, y[i], x[i], d[i]);
        float sums[2] = {0.0f, 0.0f};   // of s^2 and g s
        auto add_up = [&](float k) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                if constexpr (!KEEP) {
                    __builtin_amdgcn_sched_barrier(0);
                    load(row, i, y[0], x[0], d[0]);
                    load_weight(i);
                }
                float a[8], s[8], g[8];
                values8(y[KEEP ? i : 0], yf, a);
                values8(x[KEEP ? i : 0], xf, s);
                weight(i, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    s[e] *= k;
                    sums[0] = __builtin_fmaf(s[e], s[e], sums[0]);
                    sums[1] = __builtin_fmaf(a[e] * g[e], s[e], sums[1]);
                }
                if constexpr (FAST)
                    if (k != 1.0f)   // a power of two: bf16 holds these too
                        x[i].lo = u32x4_t{pack2(s[0], s[1]), pack2(s[2], s[3]), pack2(s[4], s[5]), pack2(s[6], s[7])};
            }
            block_sum<W>(sums, t[turn]);
        };
        add_up(1.0f);
        const float k = range_scale(sums[0], p.eps);
        if (k != 1.0f) {
            sums[0] = sums[1] = 0.0f;
            turn ^= 1;
            add_up(k);
        }
        const float rho = 1.0f / __builtin_sqrtf(sums[0] / (float)p.hidden + p.eps * k * k);
        const float back = rho * rho * (sums[1] / (float)p.hidden);   // rho mean(g n)
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if constexpr (!KEEP) {
                __builtin_amdgcn_sched_barrier(0);
                load(row, i, y[0], x[0], d[0]);
                load_weight(i);
            }
            float a[8], s[8], g[8];
            values8(y[KEEP ? i : 0], yf, a);
            values8(x[KEEP ? i : 0], xf, s);
            weight(i, g);
            if constexpr (!FAST)   // (under a branch, as below, this takes 20 registers more)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] *= k;
            if (p.part)
#pragma unroll
                for (int e = 0; e < 8; ++e) dw[i][e] = __builtin_fmaf(a[e], s[e] * rho, dw[i][e]);
            if (p.dx) {
                const uint32_t c = 8 * (i * NT + first);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = rho * (a[e] * g[e] - back * s[e]);
                if (!FAST || k != 1.0f)
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[e] *= k;
                if (p.dsum) {
                    values8(d[KEEP ? i : 0], sf, a);
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[e] += a[e];
                }
                store8(p.dx, (uint64_t)row * p.lddx + c, anew<!FAST && (CH > 1)>(left8<FAST>(p.hidden, c)), p.flags & T0G_ROWS_OUT_F32, g);
            }
        }
        if constexpr (PRE)
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                y[i] = y2[i];
                x[i] = x2[i];
                d[i] = d2[i];
            }
    }
    if (!p.part) return;
    if constexpr (R > 1) {   // the workgroup's rows' parts, in their order
        __shared__ float parts[R][64][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) parts[threadIdx.x / NT][first][e] = dw[0][e];
        __syncthreads();
        if (threadIdx.x >= NT) return;
#pragma unroll
        for (int r = 1; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) dw[0][e] += parts[r][first][e];
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = 8 * (i * NT + first);
        store8(p.part, (uint64_t)blockIdx.x * p.ldpart + c, left8<FAST>(p.hidden, c), true, dw[i]);
    }
}

// A workgroup adds up 32 columns: thread (r, g) = (tid / 8, tid % 8) every 128th row of 4 of them, then 16 threads
// 8 of these sums each, and one their 16, always in the same order.
__device__ __forceinline__ void column_sum(const T0gColSumArgs& p) {
    __shared__ f32x4_t part[128][8];
    const uint32_t g = threadIdx.x & 7u, r = threadIdx.x >> 3, c = 32 * blockIdx.x + 4 * g;
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < p.cols)   // rows of ldp values, a multiple of 8
#pragma unroll 4
        for (uint32_t i = r; i < p.n; i += 128) v += *at<const f32x4_t>(p.part + ((uint64_t)i * p.ldp + c) * 4);
    part[r][g] = v;
    __syncthreads();
    if (r < 16) {
#pragma unroll
        for (uint32_t i = 1; i < 8; ++i) v += part[r + 16 * i][g];
        part[r][g] = v;
    }
    __syncthreads();
    if (r != 0) return;
#pragma unroll
    for (uint32_t i = 1; i < 16; ++i) v += part[i][g];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (c + e < p.cols) {
            if (p.out_bf16)
                *at<__bf16>(p.out, c + e) = (__bf16)v[e];
            else
                *at<float>(p.out, c + e) = v[e];
        }
}

// ---- 8 bits with scales ----------------------------------------------------------------
// Blocks of 1 x 128: 16 lanes a block, 1 << row_shift threads a row, U rows of a thread in flight.
// FAST: bf16 in rows of whole pieces of 8.
template <bool FAST>
__device__ __forceinline__ void quantize_rows(const T0gQuantArgs& p) {
    constexpr int U = 4;
    const bool f32 = !FAST && p.flags & T0G_ROWS_X_F32, e5m2 = p.flags & T0G_ROWS_E5M2;
    const uint32_t width = 1u << p.row_shift, rows = 256u >> p.row_shift;
    const uint32_t c = 8 * (blockIdx.x * width + (threadIdx.x & (width - 1))), n = left8<FAST>(p.cols, c);
    for (uint64_t r0 = (uint64_t)blockIdx.y * U * rows; r0 < p.rows; r0 += (uint64_t)gridDim.y * U * rows) {
        Raw8 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = r0 + u * rows + (threadIdx.x >> p.row_shift);
            x[u] = load8(p.x, row * p.ldx + c, row < p.rows ? n : 0u, f32);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = r0 + u * rows + (threadIdx.x >> p.row_shift);
            float v[8];
            values8(x[u], f32, v);
            const BlockScale b = block_scale(row16_max(amax8(v)), e5m2);
            if (row < p.rows && n) {
                store_f8x8(p.q + row * p.ldq + c, n, f8x8(v, b.inv, b.rest, e5m2));
                if ((threadIdx.x & 15u) == 0) *at<float>(p.scales, (uint64_t)(c / T0G_SCALE_BLOCK) * p.ldsc + row) = b.scale;
            }
        }
    }
}

// 128 x 128 values: one scale for all of them (TILE), or one for each row and, for the transposed
// matrix, one for each column.  Thread (g, l) = (tid / 16, tid % 16) holds rows 8 g .. + 7 of columns
// 8 l .. + 7, so its part of each column is 8 bytes of the transposed matrix, which goes out through LDS
// in whole rows of 128 bytes, 8-byte piece g of row 8 l + e at piece g ^ l: with rows 144 bytes apart the 16 lanes l
// wrote to 2 groups of banks.
template <bool FAST>
__device__ __forceinline__ void quantize_tile(const T0gQuantArgs& p) {
    __shared__ float col_max[16][128], col_inv[128], col_rest[128];
    __shared__ __attribute__((aligned(16))) char out[128 * 128];
    const bool f32 = !FAST && p.flags & T0G_ROWS_X_F32, e5m2 = p.flags & T0G_ROWS_E5M2, tile = p.flags & T0G_ROWS_TILE;
    const uint32_t l = threadIdx.x & 15u, g = threadIdx.x >> 4;
    const uint32_t c0 = 128 * blockIdx.x, c = c0 + 8 * l, n = left8<FAST>(p.cols, c);
    const uint32_t tiles = (p.rows + 127) / 128;
    for (uint32_t ty = blockIdx.y; ty < tiles; ty += gridDim.y) {
        const uint32_t r0 = 128 * ty, row = r0 + 8 * g;
        Raw8 x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[i] = load8(p.x, (uint64_t)(row + i) * p.ldx + c, row + i < p.rows ? n : 0u, f32);
        float v[8][8], top[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            values8(x[i], f32, v[i]);
            top[i] = row16_max(amax8(v[i]));
        }
        float cm[8];   // the columns' largest over the thread's rows
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cm[e] = __builtin_fabsf(v[0][e]);
#pragma unroll
            for (int i = 1; i < 8; ++i) cm[e] = max_(cm[e], __builtin_fabsf(v[i][e]));
        }
        BlockScale whole = {0.0f, 0.0f, 0.0f};
        if (tile) {
            float m = top[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = max_(m, top[i]);
            if (l == 0) col_max[g][0] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max_(m, col_max[i][0]);
            whole = block_scale(m, e5m2);
            if (threadIdx.x == 0) {
                if (p.scales) *at<float>(p.scales, (uint64_t)blockIdx.x * p.ldsc + ty) = whole.scale;
                if (p.scales_t) *at<float>(p.scales_t, (uint64_t)ty * p.ldsct + blockIdx.x) = whole.scale;
            }
        }
        if (p.q)
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const BlockScale b = tile ? whole : block_scale(top[i], e5m2);
                if (row + i < p.rows && n) {
                    store_f8x8(p.q + (uint64_t)(row + i) * p.ldq + c, n, f8x8(v[i], b.inv, b.rest, e5m2));
                    if (!tile && l == 0) *at<float>(p.scales, (uint64_t)blockIdx.x * p.ldsc + row + i) = b.scale;
                }
            }
        if (p.qt) {
            if (!tile) {
#pragma unroll
                for (int e = 0; e < 8; ++e) col_max[g][8 * l + e] = cm[e];
                __syncthreads();
                if (threadIdx.x < 128) {
                    float m = col_max[0][threadIdx.x];
#pragma unroll
                    for (int i = 1; i < 16; ++i) m = max_(m, col_max[i][threadIdx.x]);
                    const BlockScale b = block_scale(m, e5m2);
                    col_inv[threadIdx.x] = b.inv;
                    col_rest[threadIdx.x] = b.rest;
                    if (c0 + threadIdx.x < p.cols) *at<float>(p.scales_t, (uint64_t)ty * p.ldsct + c0 + threadIdx.x) = b.scale;
                }
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float inv = tile ? whole.inv : col_inv[8 * l + e], rest = tile ? whole.rest : col_rest[8 * l + e];
                float u[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = v[i][e];
                *reinterpret_cast<u32x2_t*>(out + (8 * l + e) * 128 + 8 * (g ^ l)) = f8x8(u, inv, rest, e5m2);
            }
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t piece = i * 256 + threadIdx.x, tr = piece >> 3, tc = 16 * (piece & 7u);
                const uint32_t tl = tr >> 3;
                u32x4_t w = *reinterpret_cast<const u32x4_t*>(out + tr * 128 + (tc ^ 16 * (tl >> 1)));
                if (tl & 1u) w = u32x4_t{w[2], w[3], w[0], w[1]};
                if (c0 + tr >= p.cols || r0 + tc >= p.rows) continue;
                const uint64_t to = p.qt + (uint64_t)(c0 + tr) * p.ldqt + r0 + tc;
                if (r0 + tc + 16 <= p.rows) {
                    *at<u32x4_byte>(to) = w;
                    continue;
                }
                store_f8x8(to, min(p.rows - r0 - tc, 8u), u32x2_t{w[0], w[1]});
                if (r0 + tc + 8 < p.rows) store_f8x8(to + 8, min(p.rows - r0 - tc - 8, 8u), u32x2_t{w[2], w[3]});
            }
        }
        __syncthreads();   // read before the next tile overwrites it
    }
}

// ---- around the products ---------------------------------------------------------------
// a = act(g) and its derivative.  The exponential and the reciprocal are the hardware's, each
// within 2^-22, as in the GEMMs' epilogues.  A NaN passes on, into the derivative too; infinities go through the
// formula: relu gives 0 or infinity, the others NaN for -infinity and for the derivatives.
__device__ __forceinline__ void activation(uint32_t act, float g, float& a, float& slope) {
    if (act == T0G_ACT_RELU) {
        a = g < 0.0f ? 0.0f : g;
        slope = g > 0.0f ? 1.0f : g == g ? 0.0f : g;
        return;
    }
    const float k = act == T0G_ACT_GELU ? 1.702f : 1.0f;
    const float sig = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * k * g));
    a = g * sig;
    slope = __builtin_fmaf(a, k * (1.0f - sig), sig);   // k a first would leave f32's range
}

// From the kept products: dgate = dh up act'(gate), dup = dh act(gate), in bf16 as the operands of the gradients' products:
// in f32 these would leave the matrix units' bf16 rate, in two bf16 parts take twice as long.
__device__ __forceinline__ void gated_grad(const T0gGatedGradArgs& p) {
    const uint32_t per_row = (p.features + 7) / 8;
    const uint64_t pieces = (uint64_t)p.rows * per_row;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / per_row;
        const uint32_t c = 8 * (uint32_t)(i - row * per_row), n = left8(p.features, c);
        const bool f32 = p.flags & T0G_TILE_DH_F32;
        const Raw8 rd = load8(p.dh, row * p.lddh + c, n, f32), rg = load8(p.gate, row * p.ldg + c, n, false),
                   ru = load8(p.up, row * p.ldg + c, n, false);
        float d[8], g[8], u[8];
        values8(rd, f32, d);
        values8(rg, false, g);
        values8(ru, false, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float a, slope;
            activation(p.act, g[e], a, slope);
            g[e] = d[e] * u[e] * slope;
            u[e] = d[e] * a;
        }
        store8(p.c, row * p.ldc + c, n, false, g);
        store8(p.c, row * p.ldc + p.up_off + c, n, false, u);
    }
}

// Bytes [c, c + 16) of a row that ends at `end` > c, zeros past it; all loads are in the row, none waits for another.
__device__ __forceinline__ u32x4_t tail16(uint64_t row, uint32_t c, uint32_t end) {
    uint8_t b[16];
#pragma unroll
    for (uint32_t e = 0; e < 16; ++e) b[e] = *at<const uint8_t>(row, min(c + e, end - 1));
    u32x4_t w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (uint32_t e = 0; e < 16; ++e) w[e / 4] |= (c + e < end ? (uint32_t)b[e] : 0u) << (8 * (e & 3));
    return w;
}

// A wave a row, 16 bytes a lane; rows may start anywhere.
__device__ __forceinline__ void pad_rows(const T0gPadArgs& p) {
    const auto& o = p.a[blockIdx.y];
    for (uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6); row < o.rows; row += gridDim.x * 4) {
        const uint64_t from = o.src + row * o.lds, to = o.dst + row * o.ldd;
        for (uint32_t c = 16 * (threadIdx.x & 63u); c < o.ldd; c += 1024) {
            u32x4_t w = {0u, 0u, 0u, 0u};
            if (c + 16 <= o.bytes) {
                w = *at<const u32x4_byte>(from + c);
            } else if (c < o.bytes) {
                w = tail16(from, c, o.bytes);
            }
            *at<u32x4_t>(to + c) = w;
        }
    }
}

__device__ __forceinline__ void add_planes(const T0gAddArgs& p) {
    const uint32_t per_row = p.ldp / 4;
    const uint64_t pieces = (uint64_t)p.rows * per_row;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / per_row;
        const uint32_t c = 4 * (uint32_t)(i - row * per_row);
        const f32x4_t v = *at<const f32x4_t>(p.p0 + i * 16) + *at<const f32x4_t>(p.p1 + i * 16);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (c + e < p.cols) {
                if (p.out_bf16)
                    *at<__bf16>(p.out, row * p.ldo + c + e) = (__bf16)v[e];
                else
                    *at<float>(p.out, row * p.ldo + c + e) = v[e];
            }
    }
}

}  // namespace t0g

#endif
