// The feed-forward layer's calls: argument checks, kernel choice, scratch and launches.  The
// kernels are in ffn_gfx950.hip; the gated pair's gradients are products of the library's own GEMMs.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <initializer_list>
#include <mutex>
#include <string>
#include <vector>

#include "t0g.h"
#include "t0g_internal.h"
#include "t0g_kernel_args.h"

namespace t0g {

namespace {

// Limits of the kernels' 32-bit offsets within a tile of 256 rows: bytes of a row, and rows and
// columns of an array.
constexpr uint64_t kMaxRowBytes = (1ull << 31) / 256 - 128;
constexpr uint32_t kMaxRows = 0x7FFFFFFFu;
constexpr uint32_t kMaxGridY = 65535;

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }
bool is_float(uint32_t t) { return t <= T0G_BF16; }
bool is_f8(uint32_t t) { return t == T0G_E4M3 || t == T0G_E5M2; }
uint32_t size_of(uint32_t t) { return t == T0G_F32 ? 4 : t == T0G_BF16 ? 2 : 1; }
uint32_t blocks_of(uint32_t n) { return (n + T0G_SCALE_BLOCK - 1) / T0G_SCALE_BLOCK; }

// A call's arrays: their leading dimensions, alignment, and that no output meets another array.
class Arrays {
  public:
    int rc = T0G_OK;
    void in(const char *name, uint64_t a, uint64_t rows, uint64_t cols, uint32_t *ld, uint32_t type) {
        add(name, a, rows, cols, ld, type, false);
    }
    void out(const char *name, uint64_t a, uint64_t rows, uint64_t cols, uint32_t *ld, uint32_t type) {
        add(name, a, rows, cols, ld, type, true);
    }
    // `output` may be `input` itself: every value is read before it is written, by the same thread.
    void in_place(const char *output, const char *input) { allowed_.push_back({output, input}); }
    int check() {
        if (rc) return rc;
        for (size_t i = 0; i < list_.size(); ++i)
            for (size_t j = 0; j < list_.size(); ++j) {
                const Array &o = list_[i], &a = list_[j];
                if (!o.output || i == j || (a.output && j < i) || o.begin >= a.end || a.begin >= o.end) continue;
                if (side_by_side(o, a) || side_by_side(a, o)) continue;
                const bool same = o.begin == a.begin && o.ld == a.ld && o.size == a.size;
                bool ok = false;
                for (const auto &p : allowed_) ok = ok || (same && p.output == std::string(o.name) && p.input == std::string(a.name));
                if (!ok) return fail(T0G_ERR_INVALID_ARG, "%s overlaps %s", o.name, a.name);
            }
        return T0G_OK;
    }

  private:
    struct Array {
        const char *name;
        uint64_t begin, end, row;   // row: bytes of its values
        uint32_t ld, size;
        bool output;
    };
    struct Pair {
        const char *output, *input;
    };
    // Columns of one tensor: rows equally far apart, b's values in the gaps of a's.
    static bool side_by_side(const Array &a, const Array &b) {
        const uint64_t pitch = (uint64_t)a.ld * a.size;
        if (pitch != (uint64_t)b.ld * b.size || b.begin < a.begin) return false;
        const uint64_t at = (b.begin - a.begin) % pitch;
        return at >= a.row && at + b.row <= pitch;
    }
    std::vector<Array> list_;
    std::vector<Pair> allowed_;

    void add(const char *name, uint64_t a, uint64_t rows, uint64_t cols, uint32_t *ld, uint32_t type, bool output) {
        const uint32_t size = size_of(type);
        if (rc) return;
        if (*ld == 0) *ld = (uint32_t)cols;
        if (*ld < cols) {
            rc = fail(T0G_ERR_INVALID_ARG, "leading dimension of %s: %u < %llu", name, *ld, (unsigned long long)cols);
            return;
        }
        if (!a) return;
        if (a % size) {
            rc = fail(T0G_ERR_INVALID_ARG, "%s is not aligned to its elements of %u bytes", name, size);
            return;
        }
        const uint64_t extent = rows && cols ? ((rows - 1) * *ld + cols) * size : 0;
        if (extent > UINT64_MAX - a) {
            rc = fail(T0G_ERR_INVALID_ARG, "%s ends past the address space", name);
            return;
        }
        if (extent) list_.push_back(Array{name, a, a + extent, cols * size, *ld, size, output});
    }
};

int check_float(const char *name, uint32_t t) {
    return is_float(t) ? T0G_OK : fail(T0G_ERR_INVALID_ARG, "bad %s %u: f32 or bf16", name, t);
}
int check_f8(const char *name, uint32_t t) {
    return is_f8(t) ? T0G_OK : fail(T0G_ERR_INVALID_ARG, "bad %s %u: e4m3 or e5m2", name, t);
}

// No exception leaves a C entry.
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::exception &e) {
        return fail(T0G_ERR_OUT_OF_MEMORY, "host: %s", e.what());
    }
}

uint32_t groups_for(uint64_t items, uint32_t per_group, uint32_t most) {
    return (uint32_t)std::min<uint64_t>((items + per_group - 1) / per_group, most);
}

// ---- the norm ---------------------------------------------------------------------------
int check_norm_sizes(uint32_t rows, uint32_t hidden, float eps, float offset) {
    if (hidden == 0 || hidden > T0G_NORM_MAX || rows > kMaxRows)
        return fail(T0G_ERR_INVALID_ARG, "bad size: %u rows, hidden %u (1 to %u)", rows, hidden, T0G_NORM_MAX);
    if (!isfinite(eps) || eps < 0.0f) return fail(T0G_ERR_INVALID_ARG, "eps %g", (double)eps);
    if (!isfinite(offset)) return fail(T0G_ERR_INVALID_ARG, "weight_offset %g", (double)offset);
    return T0G_OK;
}

int check_norm(t0g_rms_norm_desc *d) {
    int rc;
    if ((rc = check_norm_sizes(d->rows, d->hidden, d->eps, d->weight_offset)) || (rc = check_float("x_dtype", d->x_dtype)) ||
        (rc = check_float("residual_dtype", d->residual_dtype)) || (rc = check_float("weight_dtype", d->weight_dtype)) ||
        (rc = check_float("sum_dtype", d->sum_dtype)) || (rc = check_float("y_dtype", d->y_dtype)) ||
        (rc = check_f8("q_dtype", d->q_dtype)))
        return rc;
    if (!d->y && !d->q && !d->sum) return fail(T0G_ERR_INVALID_ARG, "no output: y, q or sum");
    if (!d->q != !d->scales) return fail(T0G_ERR_INVALID_ARG, "q and scales go together");
    if (d->rows && !d->x) return fail(T0G_ERR_INVALID_ARG, "NULL x");
    uint32_t packed = d->hidden;
    Arrays a;
    a.in("x", d->x, d->rows, d->hidden, &d->ldx, d->x_dtype);
    a.in("residual", d->residual, d->rows, d->hidden, &d->ldr, d->residual_dtype);
    a.in("weight", d->weight, 1, d->hidden, &packed, d->weight_dtype);
    a.out("sum", d->sum, d->rows, d->hidden, &d->ldsum, d->sum_dtype);
    a.out("y", d->y, d->rows, d->hidden, &d->ldy, d->y_dtype);
    a.out("q", d->q, d->rows, d->hidden, &d->ldq, d->q_dtype);
    a.out("scales", d->scales, blocks_of(d->hidden), d->rows, &d->ldsc, T0G_F32);
    a.in_place("sum", "x");
    a.in_place("sum", "residual");
    a.in_place("y", "x");
    return a.check();
}

// Threads of a row and pieces of 8 values of a thread; threads and rows of a workgroup.  Up to 512 values a wave has
// the row to itself (gradients of 12527x205: 27 us; one row to a workgroup 105); two pieces a thread up to 8192
// leave registers for several workgroups on a CU.
struct RowShape {
    const char *suffix;
    uint32_t threads, rows;
};
RowShape row_shape(uint32_t hidden) {
    if (hidden <= 512) return {"64x1", 256, 4};
    if (hidden <= 2048) return {"256x1", 256, 1};
    if (hidden <= 4096) return {"256x2", 256, 1};
    if (hidden <= 8192) return {"512x2", 512, 1};
    return {"1024x2", 1024, 1};
}

int norm_call(t0g_device *dev, const t0g_rms_norm_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_rms_norm_desc d = *desc;
    int rc = check_norm(&d);
    if (rc) return rc;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    uint64_t scratch;
    if ((rc = ffn_begin(dev, 0, &scratch)) || d.rows == 0) return rc;
    T0gNormArgs a;
    memset(&a, 0, sizeof a);
    a.x = d.x;
    a.residual = d.residual;
    a.weight = d.weight;
    a.sum = d.sum;
    a.y = d.y;
    a.q = d.q;
    a.scales = d.scales;
    a.rows = d.rows;
    a.hidden = d.hidden;
    a.ldx = d.ldx;
    a.ldr = d.ldr;
    a.ldsum = d.ldsum;
    a.ldy = d.ldy;
    a.ldq = d.ldq;
    a.ldsc = d.ldsc;
    a.eps = d.eps;
    a.weight_offset = d.weight_offset;
    a.flags = (d.x_dtype == T0G_F32 ? T0G_ROWS_X_F32 : 0) | (d.residual_dtype == T0G_F32 ? T0G_ROWS_R_F32 : 0) |
              (d.weight_dtype == T0G_F32 ? T0G_ROWS_W_F32 : 0) | (d.sum_dtype == T0G_F32 ? T0G_ROWS_OUT_F32 : 0) |
              (d.y_dtype == T0G_F32 ? T0G_ROWS_Y_F32 : 0) | (d.q_dtype == T0G_E5M2 ? T0G_ROWS_E5M2 : 0);
    const bool fast = d.hidden % 8 == 0 && !(a.flags & T0G_ROWS_X_F32) && !(d.residual && a.flags & T0G_ROWS_R_F32) &&
                      !(d.weight && a.flags & T0G_ROWS_W_F32);
    const RowShape s = row_shape(d.hidden);
    return ffn_launch(dev, (std::string("t0g_ffn_norm_") + s.suffix + (fast ? "_fast" : "")).c_str(), groups_for(d.rows, s.rows, 1u << 20),
                      1, s.threads, &a, sizeof a);
}

int check_norm_grad(t0g_rms_norm_backward_desc *d) {
    int rc;
    if ((rc = check_norm_sizes(d->rows, d->hidden, d->eps, d->weight_offset)) || (rc = check_float("dy_dtype", d->dy_dtype)) ||
        (rc = check_float("x_dtype", d->x_dtype)) || (rc = check_float("weight_dtype", d->weight_dtype)) ||
        (rc = check_float("dsum_dtype", d->dsum_dtype)) || (rc = check_float("dx_dtype", d->dx_dtype)) ||
        (rc = check_float("dw_dtype", d->dw_dtype)))
        return rc;
    if (!d->dx && !d->dw) return fail(T0G_ERR_INVALID_ARG, "no output: dx or dw");
    if (d->rows && (!d->x || !d->dy)) return fail(T0G_ERR_INVALID_ARG, "NULL x or dy");
    uint32_t packed = d->hidden;
    Arrays a;
    a.in("dy", d->dy, d->rows, d->hidden, &d->lddy, d->dy_dtype);
    a.in("x", d->x, d->rows, d->hidden, &d->ldx, d->x_dtype);
    a.in("weight", d->weight, 1, d->hidden, &packed, d->weight_dtype);
    a.in("dsum", d->dsum, d->rows, d->hidden, &d->ldds, d->dsum_dtype);
    a.out("dx", d->dx, d->rows, d->hidden, &d->lddx, d->dx_dtype);
    a.out("dw", d->dw, 1, d->hidden, &packed, d->dw_dtype);
    a.in_place("dx", "dy");
    a.in_place("dx", "x");
    a.in_place("dx", "dsum");
    return a.check();
}

// Workgroups of the gradient kernel, each with a row of partial sums of dw.
bool norm_grad_fast(const t0g_rms_norm_backward_desc &d) {
    return d.hidden % 8 == 0 && d.x_dtype == T0G_BF16 && d.dy_dtype == T0G_BF16 && (!d.dsum || d.dsum_dtype == T0G_BF16) &&
           (!d.weight || d.weight_dtype == T0G_BF16);
}
uint32_t norm_grad_groups(const t0g_rms_norm_backward_desc &d) {
    const RowShape s = row_shape(d.hidden);
    return groups_for(d.rows, s.rows, std::max(256u, 1024 * 256 / s.threads));
}
uint32_t norm_grad_ld(const t0g_rms_norm_backward_desc &d) { return (uint32_t)round_up(d.hidden, 8); }
size_t norm_grad_scratch(const t0g_rms_norm_backward_desc &d) {
    return d.dw ? (size_t)norm_grad_groups(d) * norm_grad_ld(d) * 4 : 0;
}

int norm_grad_call(t0g_device *dev, const t0g_rms_norm_backward_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_rms_norm_backward_desc d = *desc;
    int rc = check_norm_grad(&d);
    if (rc) return rc;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    uint64_t scratch;
    if ((rc = ffn_begin(dev, norm_grad_scratch(d), &scratch))) return rc;
    const uint32_t groups = norm_grad_groups(d);
    if (d.rows) {
        T0gNormGradArgs a;
        memset(&a, 0, sizeof a);
        a.dy = d.dy;
        a.x = d.x;
        a.weight = d.weight;
        a.dsum = d.dsum;
        a.dx = d.dx;
        a.part = d.dw ? scratch : 0;
        a.rows = d.rows;
        a.hidden = d.hidden;
        a.lddy = d.lddy;
        a.ldx = d.ldx;
        a.ldds = d.ldds;
        a.lddx = d.lddx;
        a.ldpart = norm_grad_ld(d);
        a.eps = d.eps;
        a.weight_offset = d.weight_offset;
        a.flags = (d.dy_dtype == T0G_F32 ? T0G_ROWS_Y_F32 : 0) | (d.x_dtype == T0G_F32 ? T0G_ROWS_X_F32 : 0) |
                  (d.weight_dtype == T0G_F32 ? T0G_ROWS_W_F32 : 0) | (d.dsum_dtype == T0G_F32 ? T0G_ROWS_R_F32 : 0) |
                  (d.dx_dtype == T0G_F32 ? T0G_ROWS_OUT_F32 : 0);
        const bool fast = norm_grad_fast(d);
        const RowShape s = row_shape(d.hidden);
        if ((rc = ffn_launch(dev, (std::string("t0g_ffn_norm_grad_") + s.suffix + (fast ? "_fast" : "")).c_str(), groups, 1, s.threads,
                             &a, sizeof a)))
            return rc;
    }
    if (!d.dw) return ok();
    T0gColSumArgs s;
    memset(&s, 0, sizeof s);
    s.part = scratch;
    s.out = d.dw;
    s.n = groups;   // of no rows: zeros
    s.cols = d.hidden;
    s.ldp = norm_grad_ld(d);
    s.out_bf16 = d.dw_dtype == T0G_BF16;
    return ffn_launch(dev, "t0g_ffn_column_sum", (d.hidden + 31) / 32, 1, 1024, &s, sizeof s);
}

// ---- 8-bit values -----------------------------------------------------------------------
int check_quantize(t0g_fp8_quantize_desc *d) {
    int rc;
    if ((rc = check_float("x_dtype", d->x_dtype)) || (rc = check_f8("q_dtype", d->q_dtype))) return rc;
    if (d->block > T0G_BLOCK_TILE) return fail(T0G_ERR_INVALID_ARG, "bad block %u", d->block);
    if (d->cols == 0 || d->cols > (1u << 30) || d->rows > (1u << 30))
        return fail(T0G_ERR_INVALID_ARG, "bad size: %u rows, %u columns", d->rows, d->cols);
    if (!d->q && !d->qt) return fail(T0G_ERR_INVALID_ARG, "no output: q or qt");
    if (!d->q != !d->scales || !d->qt != !d->scales_t) return fail(T0G_ERR_INVALID_ARG, "8-bit values and scales go together");
    if (d->rows && !d->x) return fail(T0G_ERR_INVALID_ARG, "NULL x");
    const bool tile = d->block == T0G_BLOCK_TILE;
    Arrays a;
    a.in("x", d->x, d->rows, d->cols, &d->ldx, d->x_dtype);
    a.out("q", d->q, d->rows, d->cols, &d->ldq, d->q_dtype);
    a.out("scales", d->scales, blocks_of(d->cols), tile ? blocks_of(d->rows) : d->rows, &d->ldsc, T0G_F32);
    a.out("qt", d->qt, d->cols, d->rows, &d->ldqt, d->q_dtype);
    a.out("scales_t", d->scales_t, blocks_of(d->rows), tile ? blocks_of(d->cols) : d->cols, &d->ldsct, T0G_F32);
    return a.check();
}

int quantize_call(t0g_device *dev, const t0g_fp8_quantize_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_fp8_quantize_desc d = *desc;
    int rc = check_quantize(&d);
    if (rc) return rc;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    uint64_t scratch;
    if ((rc = ffn_begin(dev, 0, &scratch)) || d.rows == 0) return rc;
    T0gQuantArgs a;
    memset(&a, 0, sizeof a);
    a.x = d.x;
    a.q = d.q;
    a.scales = d.scales;
    a.qt = d.qt;
    a.scales_t = d.scales_t;
    a.rows = d.rows;
    a.cols = d.cols;
    a.ldx = d.ldx;
    a.ldq = d.ldq;
    a.ldsc = d.ldsc;
    a.ldqt = d.ldqt;
    a.ldsct = d.ldsct;
    a.flags = (d.x_dtype == T0G_F32 ? T0G_ROWS_X_F32 : 0) | (d.q_dtype == T0G_E5M2 ? T0G_ROWS_E5M2 : 0) |
              (d.block == T0G_BLOCK_TILE ? T0G_ROWS_TILE : 0);
    const bool fast = d.x_dtype == T0G_BF16 && d.cols % 8 == 0;
    if (d.qt || d.block == T0G_BLOCK_TILE)
        return ffn_launch(dev, fast ? "t0g_ffn_quantize_tile_fast" : "t0g_ffn_quantize_tile", blocks_of(d.cols), std::min(blocks_of(d.rows), kMaxGridY), 256, &a, sizeof a);
    const uint32_t pieces = blocks_of(d.cols) * 16;
    a.row_shift = 4;
    while (a.row_shift < 8 && (1u << a.row_shift) < pieces) ++a.row_shift;
    const uint32_t gx = (pieces + (1u << a.row_shift) - 1) >> a.row_shift, rows = 4 * (256u >> a.row_shift);
    return ffn_launch(dev, fast ? "t0g_ffn_quantize_rows_fast" : "t0g_ffn_quantize_rows", gx, groups_for(d.rows, rows, kMaxGridY), 256, &a, sizeof a);
}

// ---- operands of the tile kernels -------------------------------------------------------
// Rows of whole, aligned 16-byte pieces whose offsets in a tile fit 32 bits; others are copied to the scratch.
struct Operand {
    uint64_t addr = 0;
    uint32_t rows = 0, cols = 0, ld = 0, size = 1;
    bool copied = false;
    uint64_t at = 0;   // in the scratch
    uint32_t ldc = 0;
    void set(uint64_t a, uint32_t r, uint32_t c, uint32_t l, uint32_t s) {
        addr = a;
        rows = r;
        cols = c;
        ld = l;
        size = s;
        copied = a % 16 || (uint64_t)l * s % 16 || (uint64_t)c * s % 16 || (uint64_t)l * s > kMaxRowBytes;
        ldc = (uint32_t)(round_up((uint64_t)c * s, 128) / s);
    }
    uint64_t bytes() const { return copied ? (uint64_t)rows * ldc * size : 0; }
    uint64_t address(uint64_t base) const { return copied ? base + at : addr; }
    uint32_t pitch() const { return copied ? ldc : ld; }
};

uint64_t take(uint64_t *at, uint64_t bytes) {
    const uint64_t a = *at;
    *at += round_up(bytes, 256);
    return a;
}

// Copies those of up to three operands that need it, in one launch.
int run_pad(t0g_device *dev, std::initializer_list<const Operand *> list, uint64_t base) {
    T0gPadArgs p;
    memset(&p, 0, sizeof p);
    uint32_t n = 0, rows = 0;
    for (const Operand *o : list) {
        if (!o->copied || o->rows == 0) continue;
        auto &a = p.a[n++];
        a.src = o->addr;
        a.dst = base + o->at;
        a.lds = (uint64_t)o->ld * o->size;
        a.ldd = (uint64_t)o->ldc * o->size;
        a.rows = o->rows;
        a.bytes = o->cols * o->size;
        rows = std::max(rows, o->rows);
    }
    return n ? ffn_launch(dev, "t0g_ffn_pad_rows", groups_for(rows, 4, 1u << 16), n, 256, &p, sizeof p) : (int)T0G_OK;
}

// The K of a product of few tiles goes to several workgroups, in slices of at least kLeastStages stages (a slice's
// first loads take about as long as two stages), until kFill workgroups, two for each CU, are there; their sums go
// to f32 planes.  (64 rows of 11008x4096 in 8 bits 18 us, 64 of 4096x11008 into f32 22.)
constexpr uint32_t kFill = 2 * kNumCUs, kLeastStages = 4;
struct Slices {
    uint32_t n = 1, stages = 0, ldp = 0;
    uint64_t at = 0, bytes = 0;
    void set(uint64_t tiles, uint32_t k_stages, uint32_t m, uint32_t n_, uint32_t products) {
        stages = k_stages;
        if (tiles == 0 || tiles > kFill / 2) return;
        const uint32_t want = (uint32_t)std::min<uint64_t>(kFill / tiles, k_stages / kLeastStages);
        if (want < 2) return;
        stages = (k_stages + want - 1) / want;
        n = (k_stages + stages - 1) / stages;
        ldp = (uint32_t)round_up(n_, 4);
        bytes = (uint64_t)n * products * m * ldp * 4;
    }
};
uint64_t tiles_of(uint32_t m, uint32_t n, uint32_t bm, uint32_t bn) { return ((uint64_t)m + bm - 1) / bm * (((uint64_t)n + bn - 1) / bn); }

// Tiles of 128 rows instead of 64: both kinds run two to a CU; a round of the larger ones takes about 1.6 times as
// long (gated 1000x2731x1023, 688 tiles in two rounds or 344 in one: 28 us or 25; 8 bits 777x5001x1023, 520 or 280:
// 22 either way).
bool middle(uint32_t m, uint32_t n, uint32_t bn) {
    auto rounds = [&](uint32_t bm) { return (tiles_of(m, n, bm, bn) + 2 * kNumCUs - 1) / (2 * kNumCUs); };
    return 16 * rounds(128) < 10 * rounds(64);
}

int run_join(t0g_device *dev, const T0gTileArgs &t, const Slices &s, uint32_t gated) {
    T0gJoinArgs j;
    memset(&j, 0, sizeof j);
    j.t = t;
    j.slices = s.n;
    j.gated = gated;
    return ffn_launch(dev, "t0g_ffn_join_slices", groups_for((uint64_t)t.m * (s.ldp / 4), 256, 1u << 16), 1, 256, &j, sizeof j);
}

// Rows and columns of a kernel's tile.
struct Tile {
    uint32_t m, n;
};
// A launch has fewer than 2^32 threads, 512 of a tile at most.
int check_tiles(uint32_t m, uint32_t n, Tile tile) {
    if (tiles_of(m, n, tile.m, tile.n) < (1u << 22)) return T0G_OK;
    return fail(T0G_ERR_INVALID_ARG, "bad size: %u x %u in %llu tiles of %u x %u", m, n, (unsigned long long)tiles_of(m, n, tile.m, tile.n),
                tile.m, tile.n);
}
void set_tiles(T0gTileArgs *a, Tile tile) {
    a->tiles_m = (a->m - 1) / tile.m + 1;
    a->tiles_n = (a->n - 1) / tile.n + 1;
    a->group_m = 8;
}

// ---- the 8-bit product ------------------------------------------------------------------
int check_fp8_gemm(t0g_fp8_gemm_desc *d) {
    int rc;
    if ((rc = check_f8("a_dtype", d->a_dtype)) || (rc = check_f8("b_dtype", d->b_dtype)) || (rc = check_float("out_dtype", d->out_dtype)))
        return rc;
    if (d->b_block > T0G_BLOCK_TILE) return fail(T0G_ERR_INVALID_ARG, "bad b_block %u", d->b_block);
    // offsets into a row of scales are 32 bits, and so are a launch's threads
    if (d->k == 0 || d->k > kMaxRowBytes || d->m > (1u << 28) || d->n > (1u << 26))
        return fail(T0G_ERR_INVALID_ARG, "bad size: m %u, n %u, k %u", d->m, d->n, d->k);
    if (d->m && d->n && (!d->a || !d->b || !d->c || !d->a_scales || !d->b_scales)) return fail(T0G_ERR_INVALID_ARG, "NULL operand");
    Arrays a;
    a.in("a", d->a, d->m, d->k, &d->lda, d->a_dtype);
    a.in("b", d->b, d->n, d->k, &d->ldb, d->b_dtype);
    a.in("a_scales", d->a_scales, blocks_of(d->k), d->m, &d->ldas, T0G_F32);
    a.in("b_scales", d->b_scales, blocks_of(d->k), d->b_block == T0G_BLOCK_TILE ? blocks_of(d->n) : d->n, &d->ldbs, T0G_F32);
    a.out("c", d->c, d->m, d->n, &d->ldc, d->out_dtype);
    return a.check();
}

// Rows up to which a product is bound by reading B, which then goes straight to registers.  11008x4096 in 8 bits:
// one row 10 us (64-row tiles, two LDS stages: 40), 24 rows 17, where the tiles take 18 for 64; gated, one row
// 35 (62), 24 rows 47 (64 rows 53).
constexpr uint32_t kSkinnyRows = 32;

enum class Fp8Tile { Skinny, Small, Middle, Big };
struct Fp8Plan {
    Fp8Tile tile = Fp8Tile::Skinny;
    Operand a, b;
    Slices slices;
    uint64_t bytes = 0;
    Tile size() const { return tile == Fp8Tile::Big ? Tile{256, 256} : Tile{tile == Fp8Tile::Small ? 64u : 128u, 128}; }
};
int plan_fp8(const t0g_fp8_gemm_desc &d, Fp8Plan *p) {
    if (d.m <= kSkinnyRows || d.n == 0) return T0G_OK;
    // 8192x8192x8192: 472 to 486 us in 256x256 tiles, 709 in 128x128
    if (d.out_dtype == T0G_BF16 && tiles_of(d.m, d.n, 256, 256) >= kNumCUs)
        p->tile = Fp8Tile::Big;
    else
        p->tile = middle(d.m, d.n, 128) ? Fp8Tile::Middle : Fp8Tile::Small;
    if (int rc = check_tiles(d.m, d.n, p->size())) return rc;
    p->a.set(d.a, d.m, d.k, d.lda, 1);
    p->b.set(d.b, d.n, d.k, d.ldb, 1);
    p->a.at = take(&p->bytes, p->a.bytes());
    p->b.at = take(&p->bytes, p->b.bytes());
    p->slices.set(p->tile == Fp8Tile::Small ? tiles_of(d.m, d.n, 64, 128) : 0, blocks_of(d.k), d.m, d.n, 1);
    p->slices.at = take(&p->bytes, p->slices.bytes);
    return T0G_OK;
}

int fp8_gemm_call(t0g_device *dev, const t0g_fp8_gemm_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_fp8_gemm_desc d = *desc;
    int rc = check_fp8_gemm(&d);
    if (rc) return rc;
    Fp8Plan pl;
    if ((rc = plan_fp8(d, &pl))) return rc;
    T0gTileArgs t;
    memset(&t, 0, sizeof t);
    t.m = d.m;
    t.n = d.n;
    t.k = d.k;
    const bool skinny = pl.tile == Fp8Tile::Skinny, big = pl.tile == Fp8Tile::Big, small = pl.tile == Fp8Tile::Small;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    uint64_t base;
    if ((rc = ffn_begin(dev, pl.bytes, &base)) || d.m == 0 || d.n == 0) return rc;
    t.as = d.a_scales;
    t.bs = d.b_scales;
    t.ldas = d.ldas;
    t.ldbs = d.ldbs;
    t.c = d.c;
    t.ldc = d.ldc;
    t.flags = d.out_dtype == T0G_F32 ? T0G_TILE_OUT_F32 : 0;
    const std::string types = std::string(d.a_dtype == T0G_E4M3 ? "e4" : "e5") + (d.b_dtype == T0G_E4M3 ? "e4" : "e5") +
                              (d.b_block == T0G_BLOCK_TILE ? "_tile" : "_row");
    if (skinny) {
        t.a = d.a;
        t.b = d.b;
        t.lda = d.lda;
        t.ldb = d.ldb;
        const std::string symbol = std::string("t0g_ffn_f8_skinny") + (d.m <= 16 ? "1_" : "2_") + types;
        return ffn_launch(dev, symbol.c_str(), (d.n + 15) / 16, 1, 512, &t, sizeof t);
    }
    if ((rc = run_pad(dev, {&pl.a, &pl.b}, base))) return rc;
    set_tiles(&t, pl.size());
    t.a = pl.a.address(base);
    t.b = pl.b.address(base);
    t.lda = pl.a.pitch();
    t.ldb = pl.b.pitch();
    t.split_stages = pl.slices.stages;
    t.planes = pl.slices.n > 1 ? base + pl.slices.at : 0;
    t.ldp = pl.slices.ldp;
    const std::string symbol = (big ? "t0g_ffn_f8_256x256_" : small ? "t0g_ffn_f8_64x128_" : "t0g_ffn_f8_128x128_") + types +
                               (d.out_dtype == T0G_F32 ? "_f32" : "_bf16");
    if ((rc = ffn_launch(dev, symbol.c_str(), t.tiles_m * t.tiles_n, pl.slices.n, big ? 512 : 256, &t, sizeof t))) return rc;
    return pl.slices.n > 1 ? run_join(dev, t, pl.slices, 0) : (int)T0G_OK;
}

// ---- gated projections ------------------------------------------------------------------
int activation_code(uint32_t op, uint32_t *act) {
    switch (op) {
        case T0G_OP_SILU: *act = T0G_ACT_SILU; return T0G_OK;
        case T0G_OP_GELU: *act = T0G_ACT_GELU; return T0G_OK;
        case T0G_OP_RELU: *act = T0G_ACT_RELU; return T0G_OK;
        default: return fail(T0G_ERR_INVALID_ARG, "activation %u: silu, gelu or relu", op);
    }
}

int check_gated_sizes(uint32_t rows, uint32_t features, uint32_t hidden, uint32_t transpose) {
    if (transpose > T0G_NN) return fail(T0G_ERR_INVALID_ARG, "transpose %u: the weights are NT or NN", transpose);
    if (features == 0 || hidden == 0 || hidden > kMaxRowBytes / 2 || features > kMaxRowBytes / 2 || rows > kMaxRows)
        return fail(T0G_ERR_INVALID_ARG, "bad size: %u rows, %u features, hidden %u", rows, features, hidden);
    return T0G_OK;
}

int check_gated(t0g_gated_linear_desc *d, uint32_t *act) {
    int rc;
    if ((rc = check_gated_sizes(d->rows, d->features, d->hidden, d->transpose)) || (rc = activation_code(d->activation, act)) ||
        (rc = check_float("h_dtype", d->h_dtype)))
        return rc;
    if (d->rows && (!d->x || !d->wg || !d->wu || !d->h)) return fail(T0G_ERR_INVALID_ARG, "NULL operand");
    const bool nt = d->transpose == T0G_NT;
    const uint32_t wr = nt ? d->features : d->hidden, wc = nt ? d->hidden : d->features;
    Arrays a;
    a.in("x", d->x, d->rows, d->hidden, &d->ldx, T0G_BF16);
    a.in("wg", d->wg, wr, wc, &d->ldw, T0G_BF16);
    a.in("wu", d->wu, wr, wc, &d->ldw, T0G_BF16);
    a.out("h", d->h, d->rows, d->features, &d->ldh, d->h_dtype);
    a.out("gate", d->gate, d->rows, d->features, &d->ldg, T0G_BF16);
    a.out("up", d->up, d->rows, d->features, &d->ldg, T0G_BF16);
    return a.check();
}

// The gated tile kernels' operands.
enum class GatedTile { Skinny, Small, Middle, Big };
struct GatedPlan {
    GatedTile tile = GatedTile::Skinny;
    Operand x, wg, wu;
    Slices slices;
    Tile size() const { return tile == GatedTile::Big ? Tile{256, 128} : Tile{tile == GatedTile::Small ? 64u : 128u, 64}; }
    // grad: the kernels that give dgate and dup, which the 256x256 tile and the few rows' kernel do not.
    int set(uint64_t xa, uint64_t g, uint64_t u, uint32_t rows, uint32_t features, uint32_t hidden, uint32_t ldx, uint32_t ldw,
             uint32_t transpose, bool grad, uint64_t *at) {
        const bool nt = transpose == T0G_NT;
        if ((nt && rows <= kSkinnyRows && !grad) || rows == 0) return T0G_OK;
        x.set(xa, rows, hidden, ldx, 2);
        wg.set(g, nt ? features : hidden, nt ? hidden : features, ldw, 2);
        wu.set(u, nt ? features : hidden, nt ? hidden : features, ldw, 2);
        if (wg.copied || wu.copied) wg.copied = wu.copied = true;   // one leading dimension for both
        for (Operand *o : {&x, &wg, &wu}) o->at = take(at, o->bytes());
        if (!grad && big(rows, features, hidden, nt))
            tile = GatedTile::Big;
        else
            tile = middle(rows, features, 64) ? GatedTile::Middle : GatedTile::Small;
        if (int rc = check_tiles(rows, features, size())) return rc;
        slices.set(tile == GatedTile::Small ? tiles_of(rows, features, 64, 64) : 0, (hidden + 63) / 64, rows, features, 2);
        slices.at = take(at, slices.bytes);
        return T0G_OK;
    }
    // Whether the 256x256 tile takes it: enough tiles for all CUs, and 32-bit offsets in the operands.  2048x11008x4096
    // and its gradients: 944 to 985 us so, 1025 in 128x64 tiles.
    bool big(uint32_t rows, uint32_t features, uint32_t hidden, bool nt) const {
        const uint64_t most = 1ull << 30, ldb = wg.pitch(), wspan = (nt ? features + 256ull : hidden + 64ull) * ldb;
        const uint64_t g = wg.address(0), u = wu.address(0), apart = g < u ? u - g : g - u;   // as far apart in the scratch
        return tiles_of(rows, features, 256, 128) >= kNumCUs && (rows + 256ull) * x.pitch() < most && wspan < most && x.pitch() >= 64 &&
               (nt ? ldb >= 64 : ldb >= 256 && apart + wspan * 2 < (1ull << 31) - 4096);   // offsets out of range stay so less 3 KB
    }
};

// kind: 1 the forward call's outputs, 2 its gradient's.
int run_gated_tile(t0g_device *dev, T0gTileArgs *t, const GatedPlan &pl, uint64_t base, uint32_t transpose, uint32_t kind) {
    t->a = pl.x.address(base);
    t->b = pl.wg.address(base);
    t->b2 = pl.wu.address(base);
    t->lda = pl.x.pitch();
    t->ldb = pl.wg.pitch();
    t->split_stages = pl.slices.stages;
    t->planes = pl.slices.n > 1 ? base + pl.slices.at : 0;
    t->ldp = pl.slices.ldp;
    const bool nt = transpose == T0G_NT, big = pl.tile == GatedTile::Big, small = pl.tile == GatedTile::Small;
    set_tiles(t, pl.size());
    int rc;
    if ((rc = run_pad(dev, {&pl.x, &pl.wg, &pl.wu}, base))) return rc;
    const std::string symbol = std::string(big ? "t0g_ffn_gated_256x128" : small ? "t0g_ffn_gated_64x64" : "t0g_ffn_gated_128x64") +
                               (nt ? "_nt" : "_nn") + (kind == 2 ? "_grad" : "");
    if ((rc = ffn_launch(dev, symbol.c_str(), t->tiles_m * t->tiles_n, pl.slices.n, 256, t, sizeof *t))) return rc;
    return pl.slices.n > 1 ? run_join(dev, *t, pl.slices, kind) : (int)T0G_OK;
}

int gated_plan(const t0g_gated_linear_desc &d, GatedPlan *pl, uint64_t *bytes) {
    *bytes = 0;
    return pl->set(d.x, d.wg, d.wu, d.rows, d.features, d.hidden, d.ldx, d.ldw, d.transpose, false, bytes);
}

int gated_call(t0g_device *dev, const t0g_gated_linear_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_gated_linear_desc d = *desc;
    uint32_t act;
    int rc = check_gated(&d, &act);
    if (rc) return rc;
    GatedPlan pl;
    uint64_t bytes, base;
    if ((rc = gated_plan(d, &pl, &bytes))) return rc;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    if ((rc = ffn_begin(dev, bytes, &base)) || d.rows == 0) return rc;
    T0gTileArgs t;
    memset(&t, 0, sizeof t);
    t.c = d.h;
    t.ldc = d.ldh;
    t.gate = d.gate;
    t.up = d.up;
    t.ldg = d.ldg;
    t.m = d.rows;
    t.n = d.features;
    t.k = d.hidden;
    t.act = act;
    t.flags = d.h_dtype == T0G_F32 ? T0G_TILE_OUT_F32 : 0;
    if (pl.tile == GatedTile::Skinny) {
        t.a = d.x;
        t.b = d.wg;
        t.b2 = d.wu;
        t.lda = d.ldx;
        t.ldb = d.ldw;
        return ffn_launch(dev, d.rows <= 16 ? "t0g_ffn_gated_skinny1" : "t0g_ffn_gated_skinny2", (d.features + 15) / 16, 1, 512, &t,
                          sizeof t);
    }
    return run_gated_tile(dev, &t, pl, base, d.transpose, 1);
}

int check_gated_grad(t0g_gated_linear_backward_desc *d, uint32_t *act) {
    int rc;
    if ((rc = check_gated_sizes(d->rows, d->features, d->hidden, d->transpose)) || (rc = activation_code(d->activation, act)) ||
        (rc = check_float("dh_dtype", d->dh_dtype)) || (rc = check_float("dx_dtype", d->dx_dtype)) ||
        (rc = check_float("dw_dtype", d->dw_dtype)))
        return rc;
    if (d->reserved) return fail(T0G_ERR_INVALID_ARG, "reserved must be 0");
    if (!d->dx && !d->dwg && !d->dwu) return fail(T0G_ERR_INVALID_ARG, "no output: dx, dwg or dwu");
    if (!d->gate != !d->up) return fail(T0G_ERR_INVALID_ARG, "gate and up go together");
    if (d->rows && (!d->dh || !d->x || !d->wg || !d->wu)) return fail(T0G_ERR_INVALID_ARG, "NULL operand");
    const bool nt = d->transpose == T0G_NT;
    const uint32_t wr = nt ? d->features : d->hidden, wc = nt ? d->hidden : d->features;
    Arrays a;
    a.in("dh", d->dh, d->rows, d->features, &d->lddh, d->dh_dtype);
    a.in("x", d->x, d->rows, d->hidden, &d->ldx, T0G_BF16);
    a.in("wg", d->wg, wr, wc, &d->ldw, T0G_BF16);
    a.in("wu", d->wu, wr, wc, &d->ldw, T0G_BF16);
    a.in("gate", d->gate, d->rows, d->features, &d->ldg, T0G_BF16);
    a.in("up", d->up, d->rows, d->features, &d->ldg, T0G_BF16);
    a.out("dx", d->dx, d->rows, d->hidden, &d->lddx, d->dx_dtype);
    a.out("dwg", d->dwg, wr, wc, &d->lddw, d->dw_dtype);
    a.out("dwu", d->dwu, wr, wc, &d->lddw, d->dw_dtype);
    return a.check();
}

// Products that add up to one output.
struct Sum {
    uint64_t out;
    uint32_t rows, cols, ld, dtype;
    std::vector<t0g_gemm_desc> terms;
    uint64_t plane() const { return (uint64_t)rows * ldp() * 4; }
    uint32_t ldp() const { return (uint32_t)round_up(cols, 4); }
};
// The gradients' products on D = [dg | du], [rows][2 features rounded up to 8 each].
struct GatedGradPlan {
    GatedPlan tiles;                 // without the kept products
    std::vector<Sum> sums;           // addresses in the scratch are offsets from its start
    uint32_t half = 0, ldd = 0;
    uint64_t d = 0, p0 = 0, p1 = 0, ws = 0, ws_bytes = 0, bytes = 0;   // p0, p1: f32 planes of sums of several terms
};

t0g_gemm_desc product(uint64_t a, uint64_t b, uint64_t c, uint32_t m, uint32_t n, uint32_t k, uint32_t lda, uint32_t ldb,
                      uint32_t ldc, uint32_t transpose, uint32_t dtype) {
    t0g_gemm_desc g;
    memset(&g, 0, sizeof g);
    g.a = a;
    g.b = b;
    g.c = c;
    g.m = m;
    g.n = n;
    g.k = k;
    g.lda = lda;
    g.ldb = ldb;
    g.ldc = ldc;
    g.transpose = transpose;
    g.out_dtype = dtype;
    return g;
}

// No card holds operands of more pieces: one is 1 GiB or more.
constexpr uint64_t kMostPieces = 1u << 15;
// pieces: every operand below 2^30 elements, by fewer rows of it at a time.
int plan_products(const t0g_gated_linear_backward_desc &d, uint64_t base, bool pieces, GatedGradPlan *pl) {
    const bool nt = d.transpose == T0G_NT;
    const uint32_t f = d.features, es = size_of(d.dw_dtype);
    uint64_t at = 0;
    if (!d.gate)
        if (int rc = pl->tiles.set(d.x, d.wg, d.wu, d.rows, f, d.hidden, d.ldx, d.ldw, d.transpose, true, &at)) return rc;
    pl->half = (uint32_t)round_up(f, 8);
    pl->ldd = 2 * pl->half;
    pl->d = take(&at, (uint64_t)d.rows * pl->ldd * 2);
    const uint64_t dg = base + pl->d, du = dg + (uint64_t)pl->half * 2;
    const bool whole = pl->half == f;
    const uint64_t step = nt ? (uint64_t)f * d.ldw : f;
    const bool w_stacked = whole && d.wu == d.wg + step * 2 && (nt || d.ldw >= 2 * f);
    // Rows of a piece.  One row alone may be followed by anything: its leading dimension is then its length.
    auto fit = [&](uint32_t rows, uint32_t ld) {
        const uint32_t most = ((1u << 30) - 1) / ld;
        return pieces ? std::min(rows, most >= 64 ? most / 64 * 64 : std::max(1u, most)) : rows;
    };
    auto pitch = [&](uint32_t rows, uint32_t ld, uint32_t cols) { return pieces && rows == 1 ? cols : ld; };
    auto parts = [](uint64_t n, uint32_t step) { return n ? (n - 1) / step + 1 : 0; };
    const uint64_t d_parts = parts(d.rows, fit(d.rows, pl->ldd)), w_rows = nt ? f : d.hidden;
    if (d_parts * parts(w_rows, fit((uint32_t)w_rows, d.ldw)) > kMostPieces || parts(d.rows, fit(d.rows, d.ldx)) > kMostPieces)
        return fail(T0G_ERR_INVALID_ARG, "bad size: %u rows, %u features, hidden %u with rows %u and %u apart", d.rows, f, d.hidden, d.ldx, d.ldw);
    if (d.dx) {
        struct Pair {
            uint64_t d, w;
            uint32_t k;
        };
        std::vector<Pair> pairs = {{dg, d.wg, w_stacked ? 2 * f : f}};
        if (!w_stacked) pairs.push_back({du, d.wu, f});
        const uint32_t rows = fit(d.rows, pl->ldd), cols = nt ? d.hidden : fit(d.hidden, d.ldw);
        for (uint32_t r0 = 0; r0 < d.rows; r0 += rows)
            for (uint32_t c0 = 0; c0 < d.hidden; c0 += cols) {
                const uint32_t r = std::min(rows, d.rows - r0), c = std::min(cols, d.hidden - c0);
                Sum s{d.dx + ((uint64_t)r0 * d.lddx + c0) * size_of(d.dx_dtype), r, c, d.lddx, d.dx_dtype, {}};
                for (const Pair &p : pairs) {
                    const uint32_t ks = nt ? fit(p.k, d.ldw) : p.k;
                    for (uint32_t k0 = 0; k0 < p.k; k0 += ks) {
                        const uint32_t k = std::min(ks, p.k - k0);
                        const uint64_t from = p.d + ((uint64_t)r0 * pl->ldd + k0) * 2;
                        s.terms.push_back(nt ? product(from, p.w + (uint64_t)k0 * d.ldw * 2, s.out, r, c, k, pl->ldd, pitch(k, d.ldw, c), d.lddx,
                                                       T0G_NN, d.dx_dtype)
                                             : product(from, p.w + (uint64_t)c0 * d.ldw * 2, s.out, r, c, k, pl->ldd, pitch(c, d.ldw, k), d.lddx,
                                                       T0G_NT, d.dx_dtype));
                    }
                }
                pl->sums.push_back(s);
            }
    }
    auto dw = [&](uint64_t from, uint64_t to, uint32_t features) {
        Sum s{to, nt ? features : d.hidden, nt ? d.hidden : features, d.lddw, d.dw_dtype, {}};
        const uint32_t rows = std::min(fit(d.rows, pl->ldd), fit(d.rows, d.ldx));
        uint32_t r0 = 0;
        do {   // over no rows: one product, zeros
            const uint32_t r = std::min(rows, d.rows - r0), ldx = pitch(r, d.ldx, d.hidden);
            const uint64_t dr = from + (uint64_t)r0 * pl->ldd * 2, x = d.x + (uint64_t)r0 * d.ldx * 2;
            s.terms.push_back(nt ? product(dr, x, to, features, d.hidden, r, pl->ldd, ldx, d.lddw, T0G_TN, d.dw_dtype)
                                 : product(x, dr, to, d.hidden, features, r, ldx, pl->ldd, d.lddw, T0G_TN, d.dw_dtype));
            r0 += r;
        } while (r0 < d.rows);
        pl->sums.push_back(s);
    };
    const uint64_t out_step = nt ? (uint64_t)f * d.lddw : f;
    if (whole && d.dwg && d.dwu == d.dwg + out_step * es && (nt || d.lddw >= 2 * f)) {
        dw(dg, d.dwg, 2 * f);
    } else {
        if (d.dwg) dw(dg, d.dwg, f);
        if (d.dwu) dw(du, d.dwu, f);
    }
    uint64_t plane = 0;
    for (const Sum &s : pl->sums)
        if (s.terms.size() > 1) plane = std::max(plane, s.plane());
    pl->p0 = take(&at, plane);
    pl->p1 = take(&at, plane);
    for (Sum &s : pl->sums)
        for (t0g_gemm_desc &g : s.terms) {
            if (s.terms.size() > 1) {
                g.c = base + (&g == &s.terms[0] ? pl->p0 : pl->p1);
                g.ldc = s.ldp();
                g.out_dtype = T0G_F32;
            }
            if (!d.rows) continue;
            size_t bytes = 0;
            int rc = losses_gemm_workspace(&g, false, &bytes);
            if (rc) return rc;
            pl->ws_bytes = std::max<uint64_t>(pl->ws_bytes, bytes);
        }
    pl->ws = take(&at, pl->ws_bytes);
    pl->bytes = at;
    return T0G_OK;
}

// The plan for a scratch at `base` (0: sizes only; the GEMMs' choice does not depend on it but for its alignment).  The GEMMs
// take operands of whole 16-byte pieces at most sizes, and others (an odd number of features makes D one) below 2^31
// elements: where they refuse the whole, it goes in pieces.
int plan_gated_grad(const t0g_gated_linear_backward_desc &d, uint64_t base, GatedGradPlan *pl) {
    int rc = plan_products(d, base, false, pl);
    if (rc == T0G_ERR_INVALID_ARG) {
        *pl = GatedGradPlan();
        rc = plan_products(d, base, true, pl);
    }
    return rc;
}

int gated_grad_call(t0g_device *dev, const t0g_gated_linear_backward_desc *desc) {
    if (!desc) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
    t0g_gated_linear_backward_desc d = *desc;
    uint32_t act;
    int rc = check_gated_grad(&d, &act);
    if (rc) return rc;
    uint64_t base = 0;
    GatedGradPlan sizes, pl;
    if ((rc = plan_gated_grad(d, 0, &sizes))) return rc;
    if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
    std::lock_guard<std::mutex> lk(device_mutex(dev));
    if ((rc = ffn_begin(dev, sizes.bytes, &base)) || (rc = plan_gated_grad(d, base, &pl))) return rc;
    if (d.rows && d.gate) {
        T0gGatedGradArgs g;
        memset(&g, 0, sizeof g);
        g.dh = d.dh;
        g.gate = d.gate;
        g.up = d.up;
        g.c = base + pl.d;
        g.rows = d.rows;
        g.features = d.features;
        g.lddh = d.lddh;
        g.ldg = d.ldg;
        g.ldc = pl.ldd;
        g.up_off = pl.half;
        g.flags = d.dh_dtype == T0G_F32 ? T0G_TILE_DH_F32 : 0;
        g.act = act;
        const uint64_t pieces = (uint64_t)d.rows * ((d.features + 7) / 8);
        if ((rc = ffn_launch(dev, "t0g_ffn_gated_grad", groups_for(pieces, 256, 1u << 16), 1, 256, &g, sizeof g))) return rc;
    } else if (d.rows) {
        T0gTileArgs t;
        memset(&t, 0, sizeof t);
        t.c = base + pl.d;
        t.ldc = pl.ldd;
        t.up_off = pl.half;
        t.dh = d.dh;
        t.lddh = d.lddh;
        t.m = d.rows;
        t.n = d.features;
        t.k = d.hidden;
        t.act = act;
        t.flags = d.dh_dtype == T0G_F32 ? T0G_TILE_DH_F32 : 0;
        if ((rc = run_gated_tile(dev, &t, pl.tiles, base, d.transpose, 2))) return rc;
    }
    auto run = [&](t0g_gemm_desc g) {
        g.workspace = base + pl.ws;
        g.workspace_bytes = pl.ws_bytes;
        return losses_gemm(dev, &g, false);
    };
    for (const Sum &sum : pl.sums)
        for (size_t i = 0; i < sum.terms.size(); ++i) {
            if ((rc = run(sum.terms[i]))) return rc;
            if (i == 0) continue;
            // the first term's plane takes the others', and the last sum goes out
            const bool last = i + 1 == sum.terms.size();
            T0gAddArgs a;
            memset(&a, 0, sizeof a);
            a.p0 = base + pl.p0;
            a.p1 = base + pl.p1;
            a.out = last ? sum.out : a.p0;
            a.rows = sum.rows;
            a.cols = sum.cols;
            a.ldp = sum.ldp();
            a.ldo = last ? sum.ld : a.ldp;
            a.out_bf16 = last && sum.dtype == T0G_BF16;
            if ((rc = ffn_launch(dev, "t0g_ffn_add_planes", groups_for((uint64_t)a.rows * (a.ldp / 4), 256, 1u << 16), 1, 256, &a, sizeof a)))
                return rc;
        }
    return ok();
}

}  // namespace
}  // namespace t0g

extern "C" {

int t0g_rms_norm(t0g_device *dev, const t0g_rms_norm_desc *desc) {
    return t0g::guarded([&] { return t0g::norm_call(dev, desc); });
}

int t0g_rms_norm_backward(t0g_device *dev, const t0g_rms_norm_backward_desc *desc) {
    return t0g::guarded([&] { return t0g::norm_grad_call(dev, desc); });
}

int t0g_rms_norm_backward_scratch_size(const t0g_rms_norm_backward_desc *desc, size_t *bytes) {
    return t0g::guarded([&] {
        if (!desc || !bytes) return t0g::fail(T0G_ERR_INVALID_ARG, "NULL argument");
        *bytes = 0;
        t0g_rms_norm_backward_desc d = *desc;
        int rc = t0g::check_norm_grad(&d);
        if (rc) return rc;
        *bytes = t0g::norm_grad_scratch(d);
        return t0g::ok();
    });
}

int t0g_fp8_quantize(t0g_device *dev, const t0g_fp8_quantize_desc *desc) {
    return t0g::guarded([&] { return t0g::quantize_call(dev, desc); });
}

int t0g_fp8_gemm(t0g_device *dev, const t0g_fp8_gemm_desc *desc) {
    return t0g::guarded([&] { return t0g::fp8_gemm_call(dev, desc); });
}

int t0g_fp8_gemm_scratch_size(const t0g_fp8_gemm_desc *desc, size_t *bytes) {
    return t0g::guarded([&] {
        if (!desc || !bytes) return t0g::fail(T0G_ERR_INVALID_ARG, "NULL argument");
        *bytes = 0;
        t0g_fp8_gemm_desc d = *desc;
        int rc = t0g::check_fp8_gemm(&d);
        if (rc) return rc;
        t0g::Fp8Plan pl;
        if ((rc = t0g::plan_fp8(d, &pl))) return rc;
        *bytes = pl.bytes;
        return t0g::ok();
    });
}

int t0g_gated_linear(t0g_device *dev, const t0g_gated_linear_desc *desc) {
    return t0g::guarded([&] { return t0g::gated_call(dev, desc); });
}

int t0g_gated_linear_scratch_size(const t0g_gated_linear_desc *desc, size_t *bytes) {
    return t0g::guarded([&] {
        if (!desc || !bytes) return t0g::fail(T0G_ERR_INVALID_ARG, "NULL argument");
        *bytes = 0;
        t0g_gated_linear_desc d = *desc;
        uint32_t act;
        t0g::GatedPlan pl;
        uint64_t n;
        int rc = t0g::check_gated(&d, &act);
        if (rc || (rc = t0g::gated_plan(d, &pl, &n))) return rc;
        *bytes = n;
        return t0g::ok();
    });
}

int t0g_gated_linear_backward(t0g_device *dev, const t0g_gated_linear_backward_desc *desc) {
    return t0g::guarded([&] { return t0g::gated_grad_call(dev, desc); });
}

int t0g_gated_linear_backward_scratch_size(const t0g_gated_linear_backward_desc *desc, size_t *bytes) {
    return t0g::guarded([&] {
        if (!desc || !bytes) return t0g::fail(T0G_ERR_INVALID_ARG, "NULL argument");
        *bytes = 0;
        t0g_gated_linear_backward_desc d = *desc;
        uint32_t act;
        t0g::GatedGradPlan pl;
        int rc = t0g::check_gated_grad(&d, &act);
        if (rc || (rc = t0g::plan_gated_grad(d, 0, &pl))) return rc;
        *bytes = pl.bytes;
        return t0g::ok();
    });
}

}  // extern "C"
