// Losses of a projection onto a vocabulary for MI355X (gfx950): the row kernels
// around its GEMMs.  z = x W^T is taken in pieces of the vocabulary; per row the
// softmax statistics of a chunk of columns are m = max u and s = sum 2^(u - m),
// u = z k in units of log 2, and chunks are joined as
//   M = max m,  S = sum s 2^(m - M),  log2 sum 2^u = M + log2 S.
// All statistics, losses and coefficients are f32.  The logit gradients are
// rounded to bf16 once, because the products that take them on to dx and dW
// multiply bf16 operands.
#define T0G_TILES_ONLY
#include "gemm_gfx950.hip"

namespace t0g {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <class T>
using gptr = __attribute__((address_space(1))) T*;
template <class T>
__device__ __forceinline__ gptr<T> at(uint64_t base, uint64_t i = 0) {
    return reinterpret_cast<gptr<T>>((uintptr_t)base) + i;
}

constexpr float kLn2 = 0.69314718055994531f;
constexpr uint32_t kNoToken = 0xFFFFFFFFu;
constexpr int kThreads = 256;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ninf() { return -__builtin_inff(); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Over the workgroup's W waves; `t` is W floats of LDS of this call's own.
template <int W = 4>
__device__ __forceinline__ float block_max(float v, float* t) {
    v = wave_max(v);
    if ((threadIdx.x & 63u) == 0) t[threadIdx.x >> 6] = v;
    __syncthreads();
    v = t[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = __builtin_fmaxf(v, t[w]);
    return v;
}
template <int W = 4>
__device__ __forceinline__ float block_sum(float v, float* t) {
    v = wave_sum(v);
    if ((threadIdx.x & 63u) == 0) t[threadIdx.x >> 6] = v;
    __syncthreads();
    v = t[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v += t[w];
    return v;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16);
}

}  // namespace t0g

#include "losses_tile.h"

namespace t0g {

// A label or token as an index into the vocabulary, kNoToken outside it.
__device__ __forceinline__ uint32_t token_at(uint64_t base, uint64_t i, bool wide, uint32_t vocab) {
    const int64_t v = wide ? *at<const int64_t>(base, i) : (int64_t)*at<const int32_t>(base, i);
    return v >= 0 && v < (int64_t)vocab ? (uint32_t)v : kNoToken;
}

// Row `row` of x into xz, zero for an ignored row (its hidden state may hold NaN, and
// dW's product would multiply that with the row's zero gradient) and past `hidden`.
__device__ __forceinline__ void copy_row(const T0gLossArgs& p, uint32_t row, bool used, uint32_t first, uint32_t step) {
    const uint64_t to = p.xz + (uint64_t)row * p.ldxz * 2, again = to + (uint64_t)p.rows * p.ldxz * 2;
    const bool pair = p.flags & T0G_LOSS_PAIR;
    if (p.flags & T0G_LOSS_X_VEC) {
        const uint32_t n = p.hidden / 8;
        for (uint32_t i0 = first; i0 < n; i0 += 4 * step) {
            u32x4_t v[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                v[e] = u32x4_t{0u, 0u, 0u, 0u};
                if (used && i0 + e * step < n) v[e] = *at<const u32x4_t>(p.x + (uint64_t)row * p.ldx * 2, i0 + e * step);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (i0 + e * step < n) {
                    *at<u32x4_t>(to, i0 + e * step) = v[e];
                    if (pair) *at<u32x4_t>(again, i0 + e * step) = v[e];
                }
        }
    } else {
        for (uint32_t i = first; i < p.ldxz; i += step) {
            uint16_t v = 0;
            if (used && i < p.hidden) v = *at<const uint16_t>(p.x, (uint64_t)row * p.ldx + i);
            *at<uint16_t>(to, i) = v;
            if (pair) *at<uint16_t>(again, i) = v;
        }
    }
}

// What a row is compared with, and the coefficients of its gradient's sparse part.
struct RowInfo {
    uint32_t entries, label;   // the label's entry, kNoToken for none
    float cl, ct, hq;          // of the label, of the teacher's Q; sum of Q log Q
    bool taught;
    __device__ __forceinline__ bool labelled() const { return label != kNoToken; }
    __device__ __forceinline__ bool used() const { return labelled() || taught; }
};
__device__ __forceinline__ float row_rate(const T0gLossArgs& p, uint32_t row) {
    return p.loss_scale * (p.dloss ? *at<const float>(p.dloss, row) : 1.0f) * p.logit_scale;
}
__device__ __forceinline__ uint32_t row_label(const T0gLossArgs& p, uint32_t row) {
    return p.labels ? token_at(p.labels, row, p.flags & T0G_LOSS_LABEL64, p.vocab) : kNoToken;
}
__device__ __forceinline__ RowInfo row_info(const T0gLossArgs& p, uint32_t row) {
    if (p.flags & T0G_LOSS_DIRECT) {
        const bool has = row_label(p, row) != kNoToken;
        return RowInfo{has ? 1u : 0u, has ? 0u : kNoToken, has ? p.label_weight * row_rate(p, row) : 0.0f, 0.0f, 0.0f, false};
    }
    const u32x2_t ent = *at<const u32x2_t>(p.row_ent, row);
    const f32x4_t sub = *at<const f32x4_t>(p.row_sub, row);
    return RowInfo{ent[0], ent[1], sub[0], sub[1], sub[2], sub[3] != 0.0f};
}
__device__ __forceinline__ uint32_t entry_token(const T0gLossArgs& p, uint32_t row, uint32_t e) {
    return (p.flags & T0G_LOSS_DIRECT) ? row_label(p, row) : *at<const uint32_t>(p.ent_tok, (uint64_t)row * p.slots + e);
}
__device__ __forceinline__ float entry_q(const T0gLossArgs& p, uint32_t row, uint32_t e) {
    return (p.flags & T0G_LOSS_DIRECT) ? 0.0f : *at<const float>(p.ent_q, (uint64_t)row * p.slots + e);
}
__device__ __forceinline__ float entry_z(const T0gLossArgs& p, uint32_t row, uint32_t e) {
    return (p.flags & T0G_LOSS_Z) ? *at<const float>(p.z, (uint64_t)row * p.ldz + entry_token(p, row, e))
                                  : *at<const float>(p.ent_z, (uint64_t)row * p.slots + e);
}
// l0, l1, c0, c1 of a row's gradient.  With one softmax c1 is not a coefficient but whether the row has a
// gradient: its label's and teacher's coefficients may cancel in c0, and its entries remain.
__device__ __forceinline__ f32x4_t row_params(const T0gLossArgs& p, const RowInfo& r, float l0, float l1) {
    if (!r.used()) return f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (p.flags & T0G_LOSS_DUAL) return f32x4_t{l0, l1, r.cl, r.ct};
    return f32x4_t{l0, l1, r.cl + r.ct, r.cl != 0.0f || r.ct != 0.0f ? 1.0f : 0.0f};
}
__device__ __forceinline__ bool has_gradient(const f32x4_t& par) { return par[2] != 0.0f || par[3] != 0.0f; }
__device__ __forceinline__ void store_loss(const T0gLossArgs& p, uint32_t row, const RowInfo& r, float l0, float l1, float zl,
                                           float kd) {
    float loss = 0.0f;
    if (r.labelled()) loss = p.label_weight * (l0 * kLn2 - zl * p.logit_scale);
    if (r.taught) loss += p.distill_weight * p.tau * p.tau * (r.hq + kd);
    *at<float>(p.loss, row) = loss;
    if (p.lse) *at<float>(p.lse, row) = r.used() ? l1 * kLn2 : 0.0f;
}

// What a row is compared with: its label and the teacher's distribution over its
// tokens, as entries sorted by token with equal tokens joined (their probabilities
// add), so that each entry is one logit.  Sorted by ranks: keys are unique (token, then
// position), so sums of equal tokens run in the order they were given.
__device__ __forceinline__ float teacher_logit(const T0gLossArgs& p, uint64_t i) {
    return (p.flags & T0G_LOSS_TEACHER16) ? (float)__builtin_bit_cast(__bf16, *at<const uint16_t>(p.teacher, i))
                                          : *at<const float>(p.teacher, i);
}
__device__ __forceinline__ void store_row(const T0gLossArgs& p, uint32_t row, uint32_t n, uint32_t label_slot, float hq,
                                          bool taught) {
    const float rate = row_rate(p, row);
    *at<u32x2_t>(p.row_ent, row) = u32x2_t{n, label_slot};
    *at<f32x4_t>(p.row_sub, row) = f32x4_t{label_slot != kNoToken ? p.label_weight * rate : 0.0f,
                                           taught ? p.distill_weight * p.tau * rate : 0.0f, hq, taught ? 1.0f : 0.0f};
}
// Q log Q of one token, 0 for none (v_log takes no denormals).
__device__ __forceinline__ float q_log_q(float q) { return q < 1.2e-38f ? 0.0f : q * (__builtin_amdgcn_logf(q) * kLn2); }

// Fewer than 64 entries: one wave a row, an entry a lane (2048 rows of 63 entries and 2048
// columns of x: 14 us, 19 us in the form below; 4752 rows of 16: 7 us against 20).
__device__ __forceinline__ void prepare_short(const T0gLossArgs& p, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63u, k = p.teacher ? p.top_k : 0u, total = k + 1;
    const uint32_t label = row_label(p, row);
    uint32_t t = kNoToken;
    float u = ninf();
    if (lane < k) {
        const uint64_t src = (uint64_t)row * p.ldt + lane;
        t = token_at(p.tokens, src, p.flags & T0G_LOSS_TOKEN64, p.vocab);
        u = teacher_logit(p, src);
        if (u == ninf()) t = kNoToken;   // no probability: not an entry
    }
    const bool entry = t != kNoToken;
    const bool taught = __ballot(entry) != 0;
    const float top = wave_max(entry ? u : ninf());
    float q = entry ? exp2_((u - top) * (1.44269504f / p.tau)) : 0.0f;
    const float sum = wave_sum(q);
    if (entry) q = q * (1.0f / sum);
    if (lane == k) t = label;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < total; ++j) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)t, (int)j);
        rank += o < t || (o == t && j < lane);
    }
    if (lane >= total) rank = lane;
    const uint32_t st = (uint32_t)__builtin_amdgcn_ds_permute((int)(rank * 4), (int)t);   // lane `rank` receives
    const float sq = __builtin_bit_cast(float, __builtin_amdgcn_ds_permute((int)(rank * 4), __builtin_bit_cast(int, q)));
    const uint32_t before = __shfl_up(st, 1);
    const bool valid = lane < total && st != kNoToken, head = valid && (lane == 0 || before != st);
    const uint64_t heads = __ballot(head), members = __ballot(valid);
    const uint32_t slot = (uint32_t)__popcll(heads & ((1ull << lane) - 1));
    // the sum of a run of equal tokens, in order
    const uint64_t later = heads & ~((2ull << lane) - 1);
    const uint32_t end = later ? (uint32_t)__builtin_ctzll(later) : (uint32_t)__popcll(members);
    float v = 0.0f;
    for (uint32_t j = 0; __ballot(head && lane + j < end) != 0; ++j) {
        const float x = __shfl(sq, (int)((lane + j) & 63u));
        if (head && lane + j < end) v += x;
    }
    if (head) {
        *at<uint32_t>(p.ent_tok, (uint64_t)row * p.slots + slot) = st;
        *at<float>(p.ent_q, (uint64_t)row * p.slots + slot) = v;
    }
    const uint32_t n = (uint32_t)__popcll(heads);
    if (n == 0 && lane == 0) *at<uint32_t>(p.ent_tok, (uint64_t)row * p.slots) = kNoToken;
    const float hq = wave_sum(head ? q_log_q(v) : 0.0f);
    const uint64_t at_label = __ballot(head && st == label && label != kNoToken);
    const uint32_t label_slot = at_label ? (uint32_t)__popcll(heads & (at_label - 1)) : kNoToken;
    if (p.ent_off) {   // entries before each block of columns: those with a smaller token
        // heads' tokens to lanes 0 .. n - 1, the others past them
        const uint32_t to = head ? slot : n + (uint32_t)__popcll(~heads & ((1ull << lane) - 1));
        const uint32_t ht = (uint32_t)__builtin_amdgcn_ds_permute((int)(to * 4), (int)(head ? st : kNoToken));
        for (uint32_t b0 = 0; b0 < p.off_ld; b0 += 64) {
            const uint32_t b = b0 + lane;
            uint32_t lo = 0;   // first lane whose token is not smaller; lane 63 is no head
#pragma unroll
            for (uint32_t half = 32; half; half >>= 1)
                if ((uint32_t)__shfl((int)ht, (int)(lo + half - 1)) < b * T0G_LOSS_BLOCK) lo += half;
            if (b < p.off_ld) *at<uint16_t>(p.ent_off, (uint64_t)row * p.off_ld + b) = (uint16_t)lo;
        }
    }
    if (lane == 0) store_row(p, row, n, label_slot, hq, taught);
    if (p.xz) copy_row(p, row, label != kNoToken || taught, lane, 64);
}

// More: a workgroup a row, its entries in LDS, sorted 64 at a time by a wave, whose entries then
// search the other 64s: 4096 rows of 129 entries 43 us, 8192 of 1025 309 (1248 comparing all
// pairs, 16 bytes of keys a read; 46 for the former).
__device__ __forceinline__ void prepare_long(const T0gLossArgs& p, uint32_t row) {
    constexpr uint32_t N = (T0G_LOSS_MAX_TOP + 1 + kThreads - 1) / kThreads * kThreads;
    __shared__ uint32_t tok[N], srt[N], wave_heads[4], label_at;
    __shared__ float q[N], sq[N];
    __shared__ float red[3][4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, k = p.top_k, total = k + 1;
    const uint32_t label = row_label(p, row);
    float top = ninf();
    for (uint32_t i = tid; i < N && i - lane < total; i += kThreads) {   // a wave's whole 64
        uint32_t t = kNoToken;
        if (i < k) {
            const uint64_t src = (uint64_t)row * p.ldt + i;
            t = token_at(p.tokens, src, p.flags & T0G_LOSS_TOKEN64, p.vocab);
            const float u = teacher_logit(p, src);
            if (u == ninf()) t = kNoToken;   // no probability: not an entry
            q[i] = u;
            if (t != kNoToken) top = __builtin_fmaxf(top, u);
        } else if (i == k) {
            t = label;
            q[i] = 0.0f;
        }
        tok[i] = t;
        srt[i] = kNoToken;
    }
    if (tid == 0) label_at = kNoToken;
    top = block_max(top, red[0]);
    float sum = 0.0f, any = 0.0f;
    const float scale = 1.44269504f / p.tau;
    for (uint32_t i = tid; i < k; i += kThreads) {
        float e = 0.0f;
        if (tok[i] != kNoToken) {
            e = exp2_((q[i] - top) * scale);
            any = 1.0f;
        }
        q[i] = e;
        sum += e;
    }
    sum = block_sum(sum, red[1]);
    any = block_max(any, red[2]);
    const bool taught = any > 0.0f;
    const float inv = taught ? 1.0f / sum : 0.0f;
    // each wave sorts its own 64s, then every entry looks up its place in the others
    uint32_t ranks[N / kThreads];
#pragma unroll
    for (uint32_t g = 0; g < N / kThreads; ++g) {
        const uint32_t i = g * kThreads + tid;
        if (i - lane >= total) break;
        const uint32_t t = tok[i];
        uint32_t r = 0;
        for (uint32_t j = 0; j < 64; ++j) {
            const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)t, (int)j);
            r += o < t || (o == t && j < lane);
        }
        tok[i - lane + r] = t;
        ranks[g] = t != kNoToken ? r : kNoToken;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t g = 0; g < N / kThreads; ++g) {
        const uint32_t i = g * kThreads + tid;
        if (i - lane >= total) break;
        if (ranks[g] == kNoToken) continue;
        const uint32_t t = tok[i - lane + ranks[g]];
        uint32_t rank = ranks[g];
        for (uint32_t c = 0; c < total; c += 64) {
            if (c == i - lane) continue;
            const uint32_t below = c < i ? t + 1 : t;   // of equal tokens those given before
            uint32_t lo = 0;
#pragma unroll
            for (uint32_t half = 32; half; half >>= 1)
                if (tok[c + lo + half - 1] < below) lo += half;
            rank += lo + (tok[c + lo] < below);
        }
        srt[rank] = t;
        sq[rank] = q[i] * inv;
    }
    __syncthreads();
    // first entries of equal tokens, numbered in order; their tokens take the place of the keys
    uint32_t n = 0;
    float part = 0.0f;
    for (uint32_t i0 = 0; i0 < total; i0 += kThreads) {
        const uint32_t i = i0 + tid;
        const bool head = i < total && srt[i] != kNoToken && (i == 0 || srt[i - 1] != srt[i]);
        const uint64_t mask = __ballot(head);
        if (lane == 0) wave_heads[wave] = (uint32_t)__popcll(mask);
        __syncthreads();
        uint32_t slot = n + (uint32_t)__popcll(mask & ((1ull << lane) - 1));
        for (uint32_t w = 0; w < wave; ++w) slot += wave_heads[w];
        n += wave_heads[0] + wave_heads[1] + wave_heads[2] + wave_heads[3];
        if (head) {
            float v = 0.0f;
            for (uint32_t j = i; j < total && srt[j] == srt[i]; ++j) v += sq[j];
            *at<uint32_t>(p.ent_tok, (uint64_t)row * p.slots + slot) = srt[i];
            *at<float>(p.ent_q, (uint64_t)row * p.slots + slot) = v;
            tok[slot] = srt[i];
            if (srt[i] == label) label_at = slot;
            part += q_log_q(v);
        }
        __syncthreads();
    }
    if (p.ent_off)   // entries before each block of columns
        for (uint32_t b = tid; b < p.off_ld; b += kThreads) {
            uint32_t lo = 0, hi = n;   // first entry at or past the block's first token
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (tok[mid] < b * T0G_LOSS_BLOCK)
                    lo = mid + 1;
                else
                    hi = mid;
            }
            *at<uint16_t>(p.ent_off, (uint64_t)row * p.off_ld + b) = (uint16_t)lo;
        }
    const float hq = block_sum(part, red[0]);
    if (tid == 0) store_row(p, row, n, label_at, hq, taught);
    if (p.xz) copy_row(p, row, label != kNoToken || taught, tid, kThreads);
    __syncthreads();
}

// n consecutive raw logits of a row in registers, N quads a thread of a workgroup of W
// waves, times k, -inf past the end; and their statistics.
template <int N, int W>
__device__ __forceinline__ void load_logits(const T0gLossArgs& p, uint64_t base, uint32_t n, f32x4_t (&v)[N]) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        const uint32_t c = (i * (64 * W) + threadIdx.x) * 4;
        v[i] = f32x4_t{ninf(), ninf(), ninf(), ninf()};
        if (c < n) v[i] = *at<const f32x4_t>(base, c / 4);   // rows are padded to whole quads
    }
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) v[i][e] = (i * (64 * W) + threadIdx.x) * 4 + e < n ? v[i][e] * p.k : ninf();
}
template <int N, int W>
__device__ __forceinline__ void reduce_logits(const T0gLossArgs& p, const f32x4_t (&v)[N], uint32_t n, float (&red)[3][W],
                                              float& m, float& s, float& s2) {
    m = ninf();
    s = s2 = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) m = __builtin_fmaxf(m, v[i][e]);
    m = block_max<W>(m, red[0]);
    const float from = m == ninf() ? 0.0f : m;   // no token left of these: sums of 0, not of 2^(-inf + inf)
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if ((i * (64 * W) + threadIdx.x) * 4 + e >= n) continue;
            s += exp2_(v[i][e] - from);
            if (p.flags & T0G_LOSS_DUAL) s2 += exp2_((v[i][e] - from) * p.r);
        }
    s = block_sum<W>(s, red[1]);
    if (p.flags & T0G_LOSS_DUAL) s2 = block_sum<W>(s2, red[2]);
}

// Statistics of one chunk of a row of raw logits, and the raw logits of the row's
// entries in it.
__device__ __forceinline__ void chunk_stats(const T0gLossArgs& p, uint32_t row, uint32_t chunk) {
    __shared__ float red[3][4];
    const uint32_t c0 = chunk * T0G_LOSS_CHUNK, tid = threadIdx.x;
    const uint64_t base = p.z + ((uint64_t)row * p.ldz + c0) * 4;
    const uint32_t n = min(T0G_LOSS_CHUNK, p.cols - c0);
    f32x4_t v[4];
    float m, s, s2;
    load_logits<4, 4>(p, base, n, v);
    reduce_logits<4, 4>(p, v, n, red, m, s, s2);
    if (tid == 0) {
        const uint64_t i = (uint64_t)(p.chunk0 + chunk) * p.rows + row;
        *at<f32x2_t>(p.part, i) = f32x2_t{m, s};
        if (p.flags & T0G_LOSS_DUAL) *at<float>(p.part2, i) = s2;
    }
    if (!(p.flags & T0G_LOSS_Z)) {
        const RowInfo r = row_info(p, row);
        for (uint32_t e = tid; e < r.entries; e += kThreads) {
            const uint32_t c = entry_token(p, row, e) - (p.v0 + c0);   // wraps below the chunk
            if (c < n) *at<float>(p.ent_z, (uint64_t)row * p.slots + e) = *at<const float>(base, c);
        }
        // before the first product with G (of a single piece, the gradient kernel does it)
        if ((p.flags & T0G_LOSS_DIRECT) && p.xz && p.v0 == 0 && chunk == 0) copy_row(p, row, r.used(), threadIdx.x, blockDim.x);
    }
    __syncthreads();
}

// A chunk's statistics onto those before: (m, s, s2) += (cm, cs, cs2).
__device__ __forceinline__ void join_chunk(const T0gLossArgs& p, float& m, float& s, float& s2, float cm, float cs,
                                           float cs2) {
    const float top = __builtin_fmaxf(m, cm);
    s = s * (m == top ? 1.0f : exp2_(m - top)) + cs * (cm == top ? 1.0f : exp2_(cm - top));
    if (p.flags & T0G_LOSS_DUAL)
        s2 = s2 * (m == top ? 1.0f : exp2_((m - top) * p.r)) + cs2 * (cm == top ? 1.0f : exp2_((cm - top) * p.r));
    m = top;
}
__device__ __forceinline__ void join_chunks(const T0gLossArgs& p, uint32_t row, uint32_t first, uint32_t step, float& m,
                                            float& s, float& s2) {
    m = ninf();
    s = s2 = 0.0f;
    for (uint32_t c = first; c < p.chunks; c += step) {
        const uint64_t i = (uint64_t)c * p.rows + row;
        const f32x2_t v = *at<const f32x2_t>(p.part, i);
        join_chunk(p, m, s, s2, v[0], v[1], (p.flags & T0G_LOSS_DUAL) ? *at<const float>(p.part2, i) : 0.0f);
    }
}
// The teacher's term of an entry of the loss.
__device__ __forceinline__ float entry_kd(const T0gLossArgs& p, float q, float z, float l1) {
    return q != 0.0f ? q * (l1 * kLn2 - z * (p.logit_scale / p.tau)) : 0.0f;
}

// Rows' chunks joined: their losses, log-sum-exps and gradient coefficients.  A workgroup
// takes 2^row_shift rows, so that a chunk's statistics of neighbouring rows are read as
// one line, with 256 >> row_shift threads on each.
__device__ __forceinline__ void combine_rows(const T0gLossArgs& p, uint32_t row0) {
    __shared__ float t0[kThreads], t1[kThreads];
    const uint32_t tid = threadIdx.x, per = kThreads >> p.row_shift;
    const uint32_t row = row0 + (tid & ((1u << p.row_shift) - 1)), part = tid >> p.row_shift;
    const bool live = row < p.rows, dual = p.flags & T0G_LOSS_DUAL;
    // threads of one row are 2^row_shift apart
    auto join = [&](float* t, float v, bool max) {
        __syncthreads();
        t[tid] = v;
        for (uint32_t o = kThreads / 2; o >> p.row_shift; o >>= 1) {
            __syncthreads();
            if (tid < o) t[tid] = max ? __builtin_fmaxf(t[tid], t[tid + o]) : t[tid] + t[tid + o];
        }
        __syncthreads();
        return t[tid & ((1u << p.row_shift) - 1)];
    };
    float m = ninf(), s = 0.0f, s2 = 0.0f;
    if (live) join_chunks(p, row, part, per, m, s, s2);   // each thread's own chunks first, in one pass
    const float top = join(t0, m, true);
    const float l0 = top + __builtin_amdgcn_logf(join(t0, s * (m == top ? 1.0f : exp2_(m - top)), false));
    float l1 = l0;
    if (dual) l1 = top * p.r + __builtin_amdgcn_logf(join(t1, s2 * (m == top ? 1.0f : exp2_((m - top) * p.r)), false));
    RowInfo r = {0, kNoToken, 0.0f, 0.0f, 0.0f, false};
    if (live) r = row_info(p, row);
    float kd = 0.0f;
    if (p.teacher) {
        if (r.taught)
            for (uint32_t e = part; e < r.entries; e += per)
                kd += entry_kd(p, entry_q(p, row, e), entry_z(p, row, e), l1);
        kd = join(t1, kd, false);
    }
    if (part == 0 && live) {
        const float zl = r.labelled() ? entry_z(p, row, r.label) : 0.0f;
        store_loss(p, row, r, l0, l1, zl, kd);
        if (p.row_par) *at<f32x4_t>(p.row_par, row) = row_params(p, r, l0, l1);
    }
    __syncthreads();
}

// The dense part of a logit's gradient, from u.
__device__ __forceinline__ float dense_grad(const T0gLossArgs& p, const f32x4_t& par, float u) {
    float g = par[2] * exp2_(u - par[0]);
    if (p.flags & T0G_LOSS_DUAL) g += par[3] * exp2_(u * p.r - par[1]);
    return g;
}

// The gradient of a row's entry e with raw logit z.
__device__ __forceinline__ float entry_grad(const T0gLossArgs& p, const RowInfo& r, const f32x4_t& par, uint32_t row,
                                            uint32_t e, float z) {
    const float g = dense_grad(p, par, z * p.k) - r.ct * entry_q(p, row, e);
    return e == r.label ? g - r.cl : g;
}

// The gradients of a row's entries in columns [c0, c0 + n) of the piece, over the dense part.
__device__ __forceinline__ void entry_grads(const T0gLossArgs& p, uint32_t row, uint32_t c0, uint32_t n,
                                            const f32x4_t& par, uint32_t first, uint32_t step) {
    const RowInfo r = row_info(p, row);
    for (uint32_t e = first; e < r.entries; e += step) {
        const uint32_t c = entry_token(p, row, e) - (p.v0 + c0);   // wraps below the range
        if (c >= n) continue;
        const float g = entry_grad(p, r, par, row, e, entry_z(p, row, e));
        const uint64_t o = (uint64_t)row * p.ldg + c0 + c;
        const __bf16 h = (__bf16)g;
        *at<__bf16>(p.g, o) = h;
        if (p.flags & T0G_LOSS_PAIR) *at<__bf16>(p.g, o + (uint64_t)p.rows * p.ldg) = (__bf16)(g - (float)h);
    }
}

// The loss of a row whose statistics are known, by the whole workgroup of W waves.
template <int W>
__device__ __forceinline__ void finish_row(const T0gLossArgs& p, const RowInfo& r, uint32_t row, float l0, float l1,
                                           float* red) {
    float kd = 0.0f;
    if (p.teacher) {
        if (r.taught)
            for (uint32_t e = threadIdx.x; e < r.entries; e += 64 * W)
                kd += entry_kd(p, entry_q(p, row, e), entry_z(p, row, e), l1);
        kd = block_sum<W>(kd, red);
    }
    if (threadIdx.x == 0) store_loss(p, row, r, l0, l1, r.labelled() ? entry_z(p, row, r.label) : 0.0f, kd);
    if ((p.flags & T0G_LOSS_DIRECT) && (p.flags & T0G_LOSS_Z) && p.xz) copy_row(p, row, r.used(), threadIdx.x, blockDim.x);
}

// Logit gradients of columns [c0, c0 + n) of a row in bf16, zero up to ng, then its entries.
template <int N, int W>
__device__ __forceinline__ void write_grads(const T0gLossArgs& p, const RowInfo& r, uint32_t row, const f32x4_t& par,
                                            const f32x4_t (&v)[N], uint32_t c0, uint32_t n, uint32_t ng) {
    const bool used = has_gradient(par);
    const uint64_t gb = p.g + ((uint64_t)row * p.ldg + c0) * 2;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        const uint32_t c = (i * (64 * W) + threadIdx.x) * 4;
        if (c >= ng) continue;
        float g[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) g[e] = used && c + e < n ? dense_grad(p, par, v[i][e]) : 0.0f;
        *at<u32x2_t>(gb, c / 4) = u32x2_t{pack2(g[0], g[1]), pack2(g[2], g[3])};
        if (p.flags & T0G_LOSS_PAIR) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) g[e] -= (float)(__bf16)g[e];
            *at<u32x2_t>(gb + (uint64_t)p.rows * p.ldg * 2, c / 4) = u32x2_t{pack2(g[0], g[1]), pack2(g[2], g[3])};
        }
    }
    __syncthreads();   // the dense part is written before its entries are replaced
    if (used) entry_grads(p, row, c0, n, par, threadIdx.x, 64 * W);
}

// One chunk of a row, by rows: the row's statistics from the chunks', its loss (the first
// chunk), and the chunk's logit gradients.
__device__ __forceinline__ void chunk_grad(const T0gLossArgs& p, uint32_t row, uint32_t chunk) {
    __shared__ float red[4][4];
    const uint32_t c0 = chunk * T0G_LOSS_CHUNK;
    const uint32_t n = min(T0G_LOSS_CHUNK, p.cols - c0);
    const bool dual = p.flags & T0G_LOSS_DUAL;
    const RowInfo r = row_info(p, row);
    f32x4_t v[4];
    float m, s, s2;
    load_logits<4, 4>(p, p.z + ((uint64_t)row * p.ldz + c0) * 4, n, v);
    join_chunks(p, row, threadIdx.x, kThreads, m, s, s2);
    const float top = block_max(m, red[0]);
    s = block_sum(s * (m == top ? 1.0f : exp2_(m - top)), red[1]);
    if (dual) s2 = block_sum(s2 * (m == top ? 1.0f : exp2_((m - top) * p.r)), red[2]);
    const float l0 = top + __builtin_amdgcn_logf(s), l1 = dual ? top * p.r + __builtin_amdgcn_logf(s2) : l0;
    if (p.v0 == 0 && chunk == 0) finish_row<4>(p, r, row, l0, l1, red[3]);
    write_grads<4, 4>(p, r, row, row_params(p, r, l0, l1), v, c0, n, min(T0G_LOSS_CHUNK, p.ldg - c0));
    __syncthreads();
}

// A whole row of up to 256 N W raw logits in the registers of one workgroup of W waves: statistics, loss
// and, if wanted, logit gradients.  Chunks with their joining in a second kernel, and this, per
// call: loss alone, 16 rows over 1000 tokens of width 256 12.1 / 8.2 us, over 8000 of 512 13.3 /
// 10.9, with gradients 31.8 / 28.8; at 32000 tokens they were level.  Four waves serve
// many rows better, sixteen a long row: 4096 rows over 1000 tokens with 16 and 4 waves
// 60.8 / 25.0 us, over 8000 121 / 68; 64 rows over 16000 with gradients 36.4 / 40.1.
template <int N, int W>
__device__ __forceinline__ void whole_row(const T0gLossArgs& p, uint32_t row) {
    __shared__ float red[3][W], last[W];
    const RowInfo r = row_info(p, row);
    f32x4_t v[N];
    float m, s, s2;
    load_logits<N, W>(p, p.z + (uint64_t)row * p.ldz * 4, p.cols, v);
    reduce_logits<N, W>(p, v, p.cols, red, m, s, s2);
    const float l0 = m + __builtin_amdgcn_logf(s);
    const float l1 = (p.flags & T0G_LOSS_DUAL) ? m * p.r + __builtin_amdgcn_logf(s2) : l0;
    finish_row<W>(p, r, row, l0, l1, last);
    if (p.g) write_grads<N, W>(p, r, row, row_params(p, r, l0, l1), v, 0, p.cols, p.ldg);
    __syncthreads();
}

// The same from the kept exponentials, in place: kept e = 2^(u - m) less a factor that
// was put in for its rounding, so e 2^(m - l0) is the probability, and with a second
// temperature e^r 2^(m r - l1).
__device__ __forceinline__ void kept_grad(const T0gLossArgs& p, uint32_t row, uint32_t chunk) {
    constexpr uint32_t kCols = 8 * kThreads;
    const uint32_t c0 = chunk * kCols, tid = threadIdx.x, c = c0 + 8 * tid;
    const f32x4_t par = *at<const f32x4_t>(p.row_par, row);
    const bool used = has_gradient(par);
    if (c < p.ldg) {
        u32x4_t w = {0u, 0u, 0u, 0u};
        if (used && c < p.cols) {
            const float m =
                (*at<const f32x2_t>(p.part, (uint64_t)(p.chunk0 + c / T0G_LOSS_BLOCK) * p.rows + row))[0] + kKeepLog2;
            const float f0 = par[2] * exp2_(m - par[0]);
            const u32x4_t e = *at<const u32x4_t>(p.g, ((uint64_t)row * p.ldg + c) / 8);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __builtin_bit_cast(float, (e[i] & 0xFFFFu) << 14);
                v[2 * i + 1] = __builtin_bit_cast(float, (e[i] & 0xFFFF0000u) >> 2);
            }
            if (p.flags & T0G_LOSS_DUAL) {
                const float f1 = par[3] * exp2_(m * p.r - par[1]);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = f0 * v[i] + f1 * exp2_(__builtin_amdgcn_logf(v[i]) * p.r);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= f0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1]);
        }
        *at<u32x4_t>(p.g, ((uint64_t)row * p.ldg + c) / 8) = w;
    }
    __syncthreads();   // the dense part is written before its entries are replaced
    if (used && c0 < p.cols) entry_grads(p, row, c0, min(kCols, p.cols - c0), par, tid, kThreads);
}

// 8 elements a thread and step.
__device__ __forceinline__ void copy_weight(const T0gLossCopyArgs& p) {
    typedef u32x4_t u32x4_2 __attribute__((aligned(2)));
    const uint32_t per_row = p.ldd / 8;
    const uint64_t total = (uint64_t)p.rows * per_row;
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (uint64_t)gridDim.x * kThreads) {
        const uint64_t row = i / per_row;
        const uint32_t c = (uint32_t)(i - row * per_row) * 8;
        const uint64_t src = p.src + (row * p.lds + c) * 2;
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (c + 8 <= p.cols) {
            v = *reinterpret_cast<gptr<const u32x4_2>>((uintptr_t)src);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (c + e < p.cols) v[e / 2] |= (uint32_t)*at<const uint16_t>(src, e) << 16 * (e & 1u);
        }
        *at<u32x4_t>(p.dst, i) = v;
    }
}

__device__ __forceinline__ void sum_planes(const T0gLossSumArgs& p) {
    const uint32_t w = p.vec ? 4 : 1, per_row = p.cols / w;
    const uint64_t total = (uint64_t)p.rows * per_row, plane = (uint64_t)p.rows * p.ldp;
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (uint64_t)gridDim.x * kThreads) {
        const uint64_t row = i / per_row;
        const uint32_t c = (uint32_t)(i - row * per_row) * w;
        const uint64_t o = row * p.ldo + c, q = row * p.ldp + c;
        if (p.vec) {
            f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (p.acc) v = *at<const f32x4_t>(p.acc, q / 4);
            for (uint32_t s0 = 0; s0 < p.n; s0 += 16) {   // sixteen planes' loads in flight
                f32x4_t x[16];
#pragma unroll
                for (uint32_t s = 0; s < 16; ++s)
                    if (s0 + s < p.n) x[s] = *at<const f32x4_t>(p.planes + (s0 + s) * plane * 4, q / 4);
#pragma unroll
                for (uint32_t s = 0; s < 16; ++s)
                    if (s0 + s < p.n) v += x[s];
            }
            if (p.out_bf16)
                *at<u32x2_t>(p.out, o / 4) = u32x2_t{pack2(v[0], v[1]), pack2(v[2], v[3])};
            else
                *at<f32x4_t>(p.out, o / 4) = v;
        } else {
            float v = p.acc ? *at<const float>(p.acc, q) : 0.0f;
            for (uint32_t s0 = 0; s0 < p.n; s0 += 16) {
                float x[16];
#pragma unroll
                for (uint32_t s = 0; s < 16; ++s)
                    if (s0 + s < p.n) x[s] = *at<const float>(p.planes, (s0 + s) * plane + q);
#pragma unroll
                for (uint32_t s = 0; s < 16; ++s)
                    if (s0 + s < p.n) v += x[s];
            }
            if (p.out_bf16)
                *at<__bf16>(p.out, o) = (__bf16)v;
            else
                *at<float>(p.out, o) = v;
        }
    }
}

template <bool STREAM, class T>
__device__ __forceinline__ void store16(uint64_t to, T v) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(v, at<T>(to));
    else
        *at<T>(to) = v;
}

// dW of few rows: C = A^T B over up to 32 KS rows, which writes far more than it reads and
// is bound by that.  A wave takes 32 x 128 of C, small tiles of which many stand at different
// points at once (128 x 128 took 45 us on 13 rows of 29888x2832, this 37).  A lane loads 2 and 8
// columns of 8 rows of the operands; pairs of rows make its fragments of 16x16x32 products, whose
// columns are 2 or 8 apart, so that the products of a fragment of A with all 8 of B's give a lane
// 8 neighbours of C's row and 16 lanes 256 contiguous bytes of bf16.  C goes past the caches where
// its rows are whole 128-byte lines (131072x4096: 197 us against 247; 29888x2832, whose rows are
// not, 67 against 37 us), and then leaves the weight in them for the next call.
template <int KS, bool STREAM>
__device__ __forceinline__ void outer(const T0gLossOuterArgs& p) {
    constexpr int CA = 2;
    constexpr uint32_t kTileM = 16 * CA;
    const uint32_t lane = threadIdx.x & 63u, l16 = lane & 15u, quad = lane >> 4;
    const uint32_t tiles_n = (p.n + 127) / 128, tiles_m = (p.m + kTileM - 1) / kTileM;
    const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= (uint64_t)tiles_m * tiles_n) return;
    const uint32_t inner = p.m_inner ? tiles_m : tiles_n, t0 = (uint32_t)(tile / inner), t1 = (uint32_t)(tile % inner);
    const uint32_t m0 = (p.m_inner ? t1 : t0) * kTileM;
    const uint32_t ma = m0 + CA * l16, nb = (p.m_inner ? t0 : t1) * 128 + 8 * l16;
    uint32_t a[KS][8];
    u32x4_t b[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t row = 32 * s + 8 * quad + i;
            a[s][i] = 0u;
            b[s][i] = u32x4_t{0u, 0u, 0u, 0u};
            if (row < p.rows && ma < p.m) a[s][i] = *at<const uint32_t>(p.a + ((uint64_t)row * p.lda + ma) * 2);
            if (row < p.rows && nb < p.n) b[s][i] = *at<const u32x4_t>(p.b + ((uint64_t)row * p.ldb + nb) * 2);
        }
    // the low (c = 0) or high half of 8 rows' words, rows in order
    auto column = [](auto word, int c) {
        const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
        u32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(word(2 * i + 1), word(2 * i), sel);
        return __builtin_bit_cast(bf16x8_t, v);
    };
    bf16x8_t fb[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int c = 0; c < 8; ++c) fb[s][c] = column([&](int i) { return b[s][i][c >> 1]; }, c);
#pragma unroll
    for (int c = 0; c < CA; ++c) {
        f32x4_t acc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bf16x8_t fa = column([&](int i) { return a[s][i]; }, c);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[s][e], acc[e], 0, 0, 0);
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t m = m0 + CA * (4 * quad + j) + c;
            if (m >= p.m) continue;
            const uint64_t i = (uint64_t)m * p.ldc + nb;
            if (p.vec && nb + 8 <= p.n) {
                if (p.out_bf16) {
                    const u32x4_t v = {pack2(acc[0][j], acc[1][j]), pack2(acc[2][j], acc[3][j]), pack2(acc[4][j], acc[5][j]),
                                       pack2(acc[6][j], acc[7][j])};
                    store16<STREAM>(p.c + i * 2, v);
                } else {
                    store16<STREAM>(p.c + i * 4, f32x4_t{acc[0][j], acc[1][j], acc[2][j], acc[3][j]});
                    store16<STREAM>(p.c + i * 4 + 16, f32x4_t{acc[4][j], acc[5][j], acc[6][j], acc[7][j]});
                }
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    if (nb + e < p.n) {
                        if (p.out_bf16)
                            *at<__bf16>(p.c, i + e) = (__bf16)acc[e][j];
                        else
                            *at<float>(p.c, i + e) = acc[e][j];
                    }
            }
        }
    }
}

}  // namespace t0g

// one wave a row
extern "C" __global__ void __launch_bounds__(256) t0g_loss_prepare(T0gLossArgs p) {
    for (uint32_t row = blockIdx.x * 4 + threadIdx.x / 64; row < p.rows; row += gridDim.x * 4) t0g::prepare_short(p, row);
}
extern "C" __global__ void __launch_bounds__(256) t0g_loss_prepare_long(T0gLossArgs p) {
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) t0g::prepare_long(p, row);
}
extern "C" __global__ void __launch_bounds__(256) t0g_loss_stats(T0gLossArgs p) {
    for (uint32_t row = blockIdx.y; row < p.rows; row += gridDim.y) t0g::chunk_stats(p, row, blockIdx.x);
}
extern "C" __global__ void __launch_bounds__(256) t0g_loss_combine(T0gLossArgs p) {
    for (uint32_t row = blockIdx.x << p.row_shift; row < p.rows; row += gridDim.x << p.row_shift) t0g::combine_rows(p, row);
}
extern "C" __global__ void __launch_bounds__(256) t0g_loss_grad(T0gLossArgs p) {
    for (uint32_t row = blockIdx.y; row < p.rows; row += gridDim.y) t0g::chunk_grad(p, row, blockIdx.x);
}
#define T0G_LOSS_ROW(N, W)                                                                             \
    extern "C" __global__ void __launch_bounds__(64 * W) t0g_loss_row_##N##x##W(T0gLossArgs p) {       \
        for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) t0g::whole_row<N, W>(p, row);  \
    }
T0G_LOSS_ROW(1, 1)
T0G_LOSS_ROW(1, 4)
T0G_LOSS_ROW(4, 4)
T0G_LOSS_ROW(8, 4)
T0G_LOSS_ROW(4, 16)
extern "C" __global__ void __launch_bounds__(256) t0g_loss_grad_kept(T0gLossArgs p) {
    for (uint32_t row = blockIdx.y; row < p.rows; row += gridDim.y) t0g::kept_grad(p, row, blockIdx.x);
}
// one wave a row
extern "C" __global__ void __launch_bounds__(256) t0g_loss_grad_entries(T0gLossArgs p) {
    for (uint32_t row = blockIdx.x * 4 + threadIdx.x / 64; row < p.rows; row += gridDim.x * 4) {
        const t0g::f32x4_t par = *t0g::at<const t0g::f32x4_t>(p.row_par, row);
        if (t0g::has_gradient(par)) t0g::entry_grads(p, row, 0, p.cols, par, threadIdx.x & 63u, 64);
    }
}
#define T0G_LOSS_GEMM(NAME, BK, KIND)                                                                             \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))                  \
        NAME(T0gLossGemmArgs a) {                                                                                 \
        t0g::loss_tile<BK, t0g::LossTile::KIND>(a);                                                               \
    }
T0G_LOSS_GEMM(t0g_loss_logits_nt, true, Stats)
T0G_LOSS_GEMM(t0g_loss_logits_nn, false, Stats)
T0G_LOSS_GEMM(t0g_loss_logits_nt_kept, true, Keep)
T0G_LOSS_GEMM(t0g_loss_logits_nn_kept, false, Keep)
T0G_LOSS_GEMM(t0g_loss_again_nt, true, Grad)
T0G_LOSS_GEMM(t0g_loss_again_nn, false, Grad)
extern "C" __global__ void __launch_bounds__(256) t0g_loss_copy_weight(T0gLossCopyArgs p) { t0g::copy_weight(p); }
extern "C" __global__ void __launch_bounds__(256) t0g_loss_sum(T0gLossSumArgs p) { t0g::sum_planes(p); }
#define T0G_LOSS_OUTER(KS, WAVES)                                                                        \
    extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES))) \
        t0g_loss_outer_##KS(T0gLossOuterArgs p) {                                                        \
        if (p.stream)                                                                                    \
            t0g::outer<KS, true>(p);                                                                     \
        else                                                                                             \
            t0g::outer<KS, false>(p);                                                                    \
    }
T0G_LOSS_OUTER(1, 4)
T0G_LOSS_OUTER(2, 3)
T0G_LOSS_OUTER(4, 2)
