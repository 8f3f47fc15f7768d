// Losses of a projection onto a vocabulary: argument checks, the pieces of the
// vocabulary, the scratch and the launches.  The kernels are in
// losses_gfx950.hip; the products are the library's own GEMMs.
//
// One call runs
//   prepare   every row's entries (label, teacher's tokens), the masked copy of x
//   pieces    z = x W_p^T, the chunks' softmax statistics, the entries' logits
//   combine   loss, log-sum-exp and gradient coefficients of every row
//   pieces    again, last first, for the gradients: G = dL/dz in bf16, dx += G W_p,
//             dW_p = G^T x
// in one of two forms:
//   fused     the statistics are taken in the logits GEMM's epilogue (losses_tile.h), which
//             for the last piece also leaves its exponentials, 16 bits each, where G goes;
//             the other pieces' logits are computed again with G in the epilogue (so are the
//             last's at a temperature that its exponentials cannot be taken to)
//   by rows   a piece's f32 logits go to the scratch and row kernels read them: products
//             of few rows, and operands that the 256x256 tile does not take
// By rows, labels alone need no preparation (each kernel reads them), and a vocabulary that
// one workgroup's registers hold takes its statistics, loss and G in one kernel.
// A weight whose rows are not whole 16-byte pieces is copied into ones that are, piece by
// piece, when there are rows enough to make up for that, or when it is too large for the
// GEMMs' unaligned kernels.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <exception>
#include <mutex>
#include <vector>

#include "t0g.h"
#include "t0g_internal.h"
#include "t0g_kernel_args.h"

namespace t0g {

namespace {

// A piece's f32 logits take this much (by rows), its logit gradients that much (fused; also
// what the kernels' 32-bit offsets reach), and f32 partial sums of dx are added up when
// they take more than kPlaneBytes.  With pieces of 0.86 GiB a step of 8192 rows and 131072
// tokens computed four logits of seven twice: 23.2 ms against 19.7.
constexpr uint64_t kPieceBytes = 256ull << 20;
constexpr uint64_t kFusedPieceBytes = 2048ull << 20;
constexpr uint64_t kPlaneBytes = 128ull << 20;
// The fused form is taken from kFusedRows rows (with gradients from more than kPairRows) and
// this many logits on.  By rows and fused, us per call: loss alone of width 512, 512 rows
// over 6000 tokens (3.1 M) 19 / 26, over 12000 (6.1 M) 28 / 26, 192 rows over 24000 (4.6 M) 27 / 25,
// over 98304 79 / 44; width 64, 384 rows over 12000 (4.6 M) 24 / 19; with gradients, width 512,
// 512 rows over 12000 69 / 74, 768 rows (9.2 M) 92 / 80, 2048 rows over 6000 (12 M) 102 / 96; width 2048,
// 384 rows over 24000 (9.2 M) 192 / 184, 4096 rows over 2048 (8.4 M) level; width 64, 8192 rows over 512 (4.2 M)
// 57 / 64.
constexpr uint32_t kFusedRows = 128;
constexpr uint64_t kFusedLogits = 5ull << 20, kFusedGradLogits = 8ull << 20;
// Teacher's entries of a row in a block of T0G_LOSS_BLOCK columns, on average, up to which
// the fused form is taken: its epilogue takes a row's entries one after another (147 of 280
// tokens, 2985 rows of width 768: 313 us fused, 71 by rows).  Few entries on average may still crowd
// in few blocks: all of a row's in its first ones, against spread evenly, 4096 rows of 131072 tokens,
// width 2048, 128 entries 5.79 ms either way; 2048 rows of 32000, 64 entries 785 us against 768; 2048 rows of
// 131072, width 1024, 1024 entries 2.30 ms against 2.07.
constexpr uint64_t kFusedEntries = 8;
// Rows up to which G goes into the products as two bf16, the rounded value and what the
// rounding left: few rows' roundings do not average out (one row's dx has the label's
// whole, up to 2^-8), and what bounds their products is the weight's bytes.
constexpr uint32_t kPairRows = 128;
// Rows from which an unaligned weight is copied, and what a copied piece takes at most.  Without
// and with the copy, width 1023: loss alone over 50001 tokens 300 rows 128 / 112 us, 512 rows 174 /
// 116, 777 rows 243 / 167; with gradients over 20001 tokens 300 rows 140 / 166, 512 rows 187 / 184,
// 777 rows 271 / 249.
constexpr uint32_t kCopyRows = 512;
constexpr uint64_t kCopyBytes = 512ull << 20;
// Temperatures T at which the kept exponentials of the labels' softmax give the teacher's as well, to the
// power 1 / T.  What is below 2^-126 of its block's maximum is lost and would be 2^(-126 / T): with T up
// to 4 all of a block's other tokens together 127 2^-31.5 < 2^-24 of the maximum's probability.  Their
// cutting, 0.7 2^-9, grows by 1 / T: from 0.5 on it stays below G's own rounding of 2^-8.  Other
// temperatures take a second product of the last piece (2048 rows of 32000 tokens, width 2048: 931 us
// against 769; 300 of 50000, width 768: 223 against 183).
constexpr float kKeepMinT = 0.5f, kKeepMaxT = 4.0f;
// Rows of a launch's y grid, at most (the kernels step through the rest).
constexpr uint32_t kMaxGridY = 65535;

std::atomic<uint32_t> g_form{T0G_LOSS_FORM_AUTO};

struct Range {
    uint64_t begin, end;
    const char *name;
};

struct Problem {
    t0g_linear_ce_desc d;                 // leading dimensions filled in
    const t0g_linear_distill_desc *t;     // the teacher, or nullptr
    uint32_t ldt;
    bool grad, dual;
};

// Bytes from the first to the last element of a [rows][cols] array with leading dimension ld.
uint64_t extent(uint64_t rows, uint64_t cols, uint64_t ld, uint64_t size) {
    return rows && cols ? ((rows - 1) * ld + cols) * size : 0;
}

uint32_t dtype_size(uint32_t t) { return t == T0G_BF16 ? 2 : 4; }
uint32_t index_size(uint32_t t) { return t == T0G_I64 ? 8 : 4; }

int check_ld(const char *name, uint32_t *ld, uint32_t cols) {
    if (*ld == 0) *ld = cols;
    if (*ld < cols) return fail(T0G_ERR_INVALID_ARG, "%s=%u < %u", name, *ld, cols);
    return T0G_OK;
}

int check_problem(const t0g_linear_ce_desc *desc, const t0g_linear_distill_desc *t, Problem *p) {
    p->d = *desc;
    p->t = t;
    t0g_linear_ce_desc &d = p->d;
    if (d.transpose > T0G_NN) return fail(T0G_ERR_INVALID_ARG, "transpose %u: the weight is NT or NN", d.transpose);
    if (d.label_type > T0G_I64) return fail(T0G_ERR_INVALID_ARG, "bad label_type %u", d.label_type);
    if (d.dx_dtype > T0G_BF16 || d.dw_dtype > T0G_BF16)
        return fail(T0G_ERR_INVALID_ARG, "bad gradient type (dx %u, dw %u)", d.dx_dtype, d.dw_dtype);
    if (d.vocab == 0 || d.hidden == 0 || d.vocab > 0x7FFFFFFFu || d.hidden > 0x7FFFFFFFu || d.rows > 0x7FFFFFFFu)
        return fail(T0G_ERR_INVALID_ARG, "bad size: %u rows, vocab %u, hidden %u", d.rows, d.vocab, d.hidden);
    if (!isfinite(d.logit_scale) || d.logit_scale <= 0.0f)
        return fail(T0G_ERR_INVALID_ARG, "logit_scale %g", (double)d.logit_scale);
    const bool nt = d.transpose == T0G_NT;
    const uint32_t wr = nt ? d.vocab : d.hidden, wc = nt ? d.hidden : d.vocab;
    int rc;
    if ((rc = check_ld("ldx", &d.ldx, d.hidden)) || (rc = check_ld("ldw", &d.ldw, wc)) ||
        (rc = check_ld("lddx", &d.lddx, d.hidden)) || (rc = check_ld("lddw", &d.lddw, wc)))
        return rc;
    if (!d.w || (d.rows && (!d.x || !d.loss))) return fail(T0G_ERR_INVALID_ARG, "NULL operand");
    if (d.rows && !t && !d.labels) return fail(T0G_ERR_INVALID_ARG, "cross entropy without labels");
    p->ldt = 0;
    if (t) {
        if (t->reserved) return fail(T0G_ERR_INVALID_ARG, "reserved must be 0");
        if (t->top_k == 0 || t->top_k > T0G_LOSS_MAX_TOP)
            return fail(T0G_ERR_INVALID_ARG, "top_k %u (1 to %u)", t->top_k, T0G_LOSS_MAX_TOP);
        if (t->teacher_dtype > T0G_BF16 || t->token_type > T0G_I64)
            return fail(T0G_ERR_INVALID_ARG, "bad teacher_dtype %u or token_type %u", t->teacher_dtype, t->token_type);
        if (!isfinite(t->temperature) || t->temperature <= 0.0f)
            return fail(T0G_ERR_INVALID_ARG, "temperature %g", (double)t->temperature);
        p->ldt = t->ldt;
        if ((rc = check_ld("ldt", &p->ldt, t->top_k))) return rc;
        if (d.rows && (!t->teacher || !t->tokens)) return fail(T0G_ERR_INVALID_ARG, "NULL teacher");
    }
    // every array on its element's alignment, and no output over another array
    std::vector<Range> in, out;
    auto add = [&](std::vector<Range> &v, const char *name, uint64_t a, uint64_t rows, uint64_t cols, uint64_t ld,
                   uint32_t size) {
        if (!a) return (int)T0G_OK;
        if (a % size) return fail(T0G_ERR_INVALID_ARG, "%s is not aligned to its elements of %u bytes", name, size);
        v.push_back(Range{a, a + extent(rows, cols, ld, size), name});
        return (int)T0G_OK;
    };
    if ((rc = add(in, "x", d.x, d.rows, d.hidden, d.ldx, 2)) || (rc = add(in, "w", d.w, wr, wc, d.ldw, 2)) ||
        (rc = add(in, "labels", d.labels, 1, d.rows, d.rows, index_size(d.label_type))) ||
        (rc = add(in, "dloss", d.dloss, 1, d.rows, d.rows, 4)) ||
        (rc = add(out, "loss", d.loss, 1, d.rows, d.rows, 4)) || (rc = add(out, "lse", d.lse, 1, d.rows, d.rows, 4)) ||
        (rc = add(out, "dx", d.dx, d.rows, d.hidden, d.lddx, dtype_size(d.dx_dtype))) ||
        (rc = add(out, "dw", d.dw, wr, wc, d.lddw, dtype_size(d.dw_dtype))))
        return rc;
    if (t && ((rc = add(in, "teacher", t->teacher, d.rows, t->top_k, p->ldt, dtype_size(t->teacher_dtype))) ||
              (rc = add(in, "tokens", t->tokens, d.rows, t->top_k, p->ldt, index_size(t->token_type)))))
        return rc;
    for (size_t i = 0; i < out.size(); ++i) {
        auto meets = [&](const Range &r) { return out[i].begin < r.end && r.begin < out[i].end; };
        for (const Range &r : in)
            if (meets(r)) return fail(T0G_ERR_INVALID_ARG, "%s overlaps %s", out[i].name, r.name);
        for (size_t j = 0; j < i; ++j)
            if (meets(out[j])) return fail(T0G_ERR_INVALID_ARG, "%s overlaps %s", out[i].name, out[j].name);
    }
    p->grad = d.dx || d.dw;
    p->dual = t && d.labels && t->temperature != 1.0f;
    return T0G_OK;
}

struct Piece {
    uint32_t v0, cols, chunk0, chunks;
};

// The pieces, and where everything is in the scratch.
struct Plan {
    std::vector<Piece> pieces;
    bool fused = false;
    bool keep = false;           // fused, gradients: the last piece's exponentials are kept
    bool copy_w = false;         // the pieces' weights are copied
    bool copy_x = false;         // products take xz instead of x
    bool direct = false;         // by rows, labels alone
    bool pair = false;           // G in two bf16, rows of g and xz twice
    bool padded = false;         // every operand's rows are whole 16-byte pieces
    uint32_t chunks = 0, slots = 0, ldxz = 0, off_ld = 0, least_ldg = 8;
    uint32_t group = 0;          // products of dx summed at a time (0: the one product writes dx)
    uint32_t splits = 1;         // pair: planes of each product and half
    uint32_t ldp = 0;
    uint64_t xz = 0, ent_tok = 0, ent_q = 0, ent_z = 0, row_ent = 0, row_sub = 0, row_par = 0, part = 0, part2 = 0,
             ent_off = 0, w = 0;
    uint64_t z = 0, g = 0, planes = 0, acc = 0, gemm_ws = 0;
    uint64_t gemm_ws_bytes = 0, bytes = 0;
};

uint32_t round_up(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// The GEMMs of a piece; addresses in the scratch are offsets from `base`.
t0g_gemm_desc gemm_of(uint64_t a, uint64_t b, uint64_t c, uint32_t m, uint32_t n, uint32_t k, uint32_t lda, uint32_t ldb,
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

// G's leading dimension; the fused form stores whole tiles.
uint32_t ld_of_g(const Plan &pl, const Piece &pc) {
    return std::max(round_up(pc.cols, pl.fused ? 256 : 8), pl.least_ldg);
}

uint64_t weight_piece(const Problem &p, uint64_t w, uint32_t v0, uint32_t ld, uint32_t size) {
    return w + (p.d.transpose == T0G_NT ? (uint64_t)v0 * ld : v0) * size;
}

// The operands of the products: a piece of the weight and its leading dimension, and x.
uint64_t w_of(const Problem &p, const Plan &pl, const Piece &pc, uint64_t base) {
    return pl.copy_w ? base + pl.w : weight_piece(p, p.d.w, pc.v0, p.d.ldw, 2);
}
uint32_t ldw_of(const Problem &p, const Plan &pl, const Piece &pc) {
    if (!pl.copy_w) return p.d.ldw;
    return p.d.transpose == T0G_NT ? round_up(p.d.hidden, 8) : round_up(pc.cols, 256);
}
uint64_t x_of(const Problem &p, const Plan &pl, uint64_t base) { return pl.copy_x ? base + pl.xz : p.d.x; }
uint32_t ldx_of(const Problem &p, const Plan &pl) { return pl.copy_x ? pl.ldxz : p.d.ldx; }

t0g_gemm_desc logits_gemm(const Problem &p, const Plan &pl, const Piece &pc, uint64_t base) {
    const t0g_linear_ce_desc &d = p.d;
    return gemm_of(x_of(p, pl, base), w_of(p, pl, pc, base), base + pl.z, d.rows, pc.cols, d.hidden, ldx_of(p, pl),
                   ldw_of(p, pl, pc), round_up(pc.cols, 4), d.transpose, T0G_F32);
}

// dx sums over a piece's tokens, a long K, with few tiles of output: K in as many slices as fill the CUs
// once.  The GEMMs' own choice takes powers of two, which leave up to half of them idle: 20 tiles of
// 407x1000x74752 took 131 us against 65, 1000x768x50048 103 against 68, and in 256x256 tiles
// 1697x1208x60624 537 against 291.  128x128 tiles while three slices fit and hold 12 stages of 64
// each (over 60 sizes 0.50 to 1.02 of the own choice's time, but for 568x304x123912 with 1.14; slices
// of 3 to 11 stages up to 1.64), from there 256x256 tiles with slices of 50 (0.54 to 1.00;
// 508x2888x31880 with 49 1.07), where their number is not one the own choice has (in 4 slices 2048x2048x32000
// took 7 us more than what it takes).  Not for the pair's products, whose planes cost more the
// more there are (64 rows, 50304 tokens: 115 us against 108).
void slice_long_k(t0g_gemm_desc *g) {
    static const t0g_gemm_config small = [] {
        t0g_gemm_config c;
        (void)t0g_config_preset("gfx950_128x128_k64", &c);
        return c;
    }();
    static const t0g_gemm_config big = [] {
        t0g_gemm_config c;
        (void)t0g_config_preset("gfx950_256x256_k64", &c);
        return c;
    }();
    auto tiles = [g](uint32_t side) { return (uint64_t)((g->m + side - 1) / side) * ((g->n + side - 1) / side); };
    const uint32_t stages = (g->k + 63) / 64;
    if (tiles(128) == 0) return;
    const uint64_t s1 = std::min<uint64_t>(kNumCUs / tiles(128), 64), s2 = kNumCUs / tiles(256);
    if (s1 >= 3 && stages >= s1 * 12) {
        g->config = &small;
        g->split_k = (uint32_t)s1;
    } else if (s1 < 3 && (s2 & (s2 - 1)) != 0 && stages >= s2 * 50) {
        g->config = &big;
        g->split_k = (uint32_t)s2;
    }
}

// dx of a piece: the output itself, or f32 plane `plane`.
t0g_gemm_desc dx_gemm(const Problem &p, const Plan &pl, const Piece &pc, uint64_t base, uint32_t plane) {
    const t0g_linear_ce_desc &d = p.d;
    const bool whole = pl.group == 0;
    t0g_gemm_desc g =
        gemm_of(base + pl.g, w_of(p, pl, pc, base),
                   whole ? d.dx : base + pl.planes + (uint64_t)plane * d.rows * pl.ldp * 4, pl.pair ? 2 * d.rows : d.rows,
                   d.hidden, pc.cols, ld_of_g(pl, pc), ldw_of(p, pl, pc), whole ? d.lddx : pl.ldp,
                   d.transpose == T0G_NT ? T0G_NN : T0G_NT, whole ? d.dx_dtype : (uint32_t)T0G_F32);
    if (!pl.pair) slice_long_k(&g);
    return g;
}

t0g_gemm_desc dw_gemm(const Problem &p, const Plan &pl, const Piece &pc, uint64_t base) {
    const t0g_linear_ce_desc &d = p.d;
    const uint64_t c = weight_piece(p, d.dw, pc.v0, d.lddw, dtype_size(d.dw_dtype));
    const uint32_t ldg = ld_of_g(pl, pc), rows = pl.pair ? 2 * d.rows : d.rows;
    return d.transpose == T0G_NT
               ? gemm_of(base + pl.g, base + pl.xz, c, pc.cols, d.hidden, rows, ldg, pl.ldxz, d.lddw, T0G_TN, d.dw_dtype)
               : gemm_of(base + pl.xz, base + pl.g, c, d.hidden, pc.cols, rows, pl.ldxz, ldg, d.lddw, T0G_TN, d.dw_dtype);
}

// dW of few rows as t0g_loss_outer_*, which writes at up to 5.5 TB/s where the GEMMs' tiles, each loading,
// multiplying and storing in turn, reach 3 to 4: 13 rows of 29888x2832 185 us for the whole call against
// 135, 32x32000x1024 77 against 70, 64 rows of 50304x768 107 against 97.  Not for small outputs (29 rows
// of 5120x192: 33.4 us against 35.8), nor for more than 32 rows where the rows of dW are the
// hidden ones (64 rows, 4096x128000: 816 us against 954).
constexpr uint64_t kOuterSize = 1ull << 22;
constexpr uint64_t kCacheBytes = 256ull << 20;
bool outer_dw(const Problem &p, const Plan &pl) {
    return pl.pair && p.d.rows <= (p.d.transpose == T0G_NT ? 64u : 32u) && (uint64_t)p.d.vocab * p.d.hidden >= kOuterSize;
}

// bounded: every product takes less of the weight than 2^30 values.
int plan_pieces(const Problem &p, bool bounded, Plan *pl) {
    const t0g_linear_ce_desc &d = p.d;
    const uint64_t rows = d.rows ? d.rows : 1;
    const bool nt = d.transpose == T0G_NT;
    const bool aligned = (d.w & 15) == 0 && d.ldw % 8 == 0 && (nt ? d.hidden : d.vocab) % 8 == 0;
    const bool x_aligned = (d.x & 15) == 0 && d.ldx % 8 == 0 && d.hidden % 8 == 0;
    pl->copy_w = (!aligned && d.rows >= kCopyRows) || (bounded && !nt);
    pl->padded = aligned || pl->copy_w;
    pl->ldxz = round_up(d.hidden, 8);
    // the GEMMs take operands past 2^30 values (here dW's) with leading dimensions of 256 and more
    if (rows * pl->ldxz >= (1ull << 30)) pl->least_ldg = 256;
    // the 256x256 tile takes 32-bit byte offsets, and rows of 256 or more of a weight
    // [hidden][vocab] (a copied piece has them)
    const uint64_t ldx = std::max(pl->ldxz, d.ldx), ldw = pl->copy_w ? pl->ldxz : d.ldw;
    const uint32_t form = g_form.load();
    const bool worth = form == T0G_LOSS_FORM_FUSED ? d.rows > 0
                       : p.grad ? d.rows > kPairRows && rows * d.vocab >= kFusedGradLogits
                              : d.rows >= kFusedRows && rows * d.vocab >= kFusedLogits;
    const bool sparse = !p.t || form == T0G_LOSS_FORM_FUSED || (uint64_t)p.t->top_k * T0G_LOSS_BLOCK <= kFusedEntries * d.vocab;
    pl->fused = form != T0G_LOSS_FORM_ROWS && worth && sparse && pl->padded && d.rows * ldx < (1ull << 30) && (d.max_piece == 0 || d.max_piece >= 256) &&
                (nt ? ldw * 256 < (1ull << 30) : pl->copy_w || (d.ldw >= 256 && d.hidden * ldw < (1ull << 30)));
    pl->keep = pl->fused && p.grad && !(p.dual && !(p.t->temperature >= kKeepMinT && p.t->temperature <= kKeepMaxT));
    // xz is dW's operand; the logits' too where x itself is not aligned like the weight, and
    // wherever it is there before them
    pl->copy_x = (pl->padded && !x_aligned) || (p.grad && (pl->fused || p.t));
    pl->direct = !pl->fused && !p.t && !pl->copy_x;
    pl->pair = !pl->fused && p.grad && d.rows <= kPairRows;
    const uint32_t chunk = pl->fused ? T0G_LOSS_BLOCK : T0G_LOSS_CHUNK;
    uint64_t width = d.vocab;
    if (!pl->fused)
        width = kPieceBytes / (rows * 4);
    else if (p.grad)
        width = kFusedPieceBytes / 2 / round_up(d.rows, 256);
    if ((pl->fused || bounded) && nt) width = std::min<uint64_t>(width, ((1ull << 30) - 1) / ldw);
    if (pl->copy_w) width = std::min<uint64_t>(width, kCopyBytes / 2 / pl->ldxz);
    width = width >= d.vocab ? round_up(d.vocab, 256) : std::max<uint64_t>(256, width / 256 * 256);
    if (d.max_piece) {
        const uint32_t step = pl->fused ? 256 : 8;
        width = std::min<uint64_t>(width, std::max(step, d.max_piece / step * step));
    }
    // fused: the last piece's exponentials are kept, so the first is the short one
    const uint64_t whole = ((uint64_t)d.vocab + 255) / 256 * 256;
    const uint64_t head = pl->fused && whole > width ? whole - (whole - 1) / width * width : width;
    for (uint32_t v0 = 0; v0 < d.vocab;) {
        const uint32_t cols = (uint32_t)std::min<uint64_t>(v0 == 0 ? head : width, d.vocab - v0);
        const uint32_t chunks = (cols + chunk - 1) / chunk;
        pl->pieces.push_back(Piece{v0, cols, pl->chunks, chunks});
        pl->chunks += chunks;
        v0 += cols;
    }
    pl->slots = 1 + (p.t ? p.t->top_k : 0);
    pl->ldp = round_up(d.hidden, 4);
    const uint64_t plane = rows * pl->ldp * 4;
    if (pl->pair)
        pl->group = d.dx ? 1 : 0;
    else if (d.dx && pl->pieces.size() > 1)
        pl->group = (uint32_t)std::min<uint64_t>(pl->pieces.size(), std::max<uint64_t>(1, kPlaneBytes / plane));

    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t a = at;
        at += (bytes + 255) & ~255ull;
        return a;
    };
    uint32_t widest = 0;
    for (const Piece &pc : pl->pieces) widest = std::max(widest, pc.cols);
    const uint64_t halves = pl->pair ? 2 : 1;
    if (pl->copy_x || p.grad) pl->xz = take(halves * rows * pl->ldxz * 2);
    if (pl->copy_w) {
        const Piece wide = {0, widest, 0, 0};
        pl->w = take((uint64_t)ldw_of(p, *pl, wide) * (nt ? widest : d.hidden) * 2);
    }
    pl->ent_tok = take(rows * pl->slots * 4);
    pl->ent_q = take(rows * pl->slots * 4);
    pl->ent_z = take(rows * pl->slots * 4);
    pl->row_ent = take(rows * 8);
    pl->row_sub = take(rows * 16);
    if (p.grad) pl->row_par = take(rows * 16);
    pl->part = take(rows * pl->chunks * 8);
    if (p.dual) pl->part2 = take(rows * pl->chunks * 4);
    if (pl->fused) {
        if (p.t) {
            pl->off_ld = pl->chunks + 1;
            pl->ent_off = take(rows * pl->off_ld * 2);
        }
        if (p.grad) pl->g = take((uint64_t)round_up(d.rows, 256) * round_up(widest, 256) * 2);
    } else {
        pl->z = take(rows * round_up(widest, 4) * 4);
        if (p.grad) pl->g = take(halves * rows * ld_of_g(*pl, Piece{0, widest, 0, 0}) * 2);
    }
    if (pl->group) {
        uint32_t splits = 1;
        if (pl->pair)
            for (const Piece &pc : pl->pieces) {
                const t0g_gemm_desc g = dx_gemm(p, *pl, pc, 0, 0);
                int rc = losses_gemm_planes_count(&g, pl->padded, &splits);
                if (rc) return rc;
                pl->splits = std::max(pl->splits, splits);
            }
        pl->planes = take(pl->group * halves * pl->splits * plane);
        if (pl->group < pl->pieces.size()) pl->acc = take(plane);
    }
    // one split-K workspace for all products, which run one after another
    for (const Piece &pc : pl->pieces) {
        t0g_gemm_desc g[3];
        int n = 0, rc;
        if (!pl->fused) g[n++] = logits_gemm(p, *pl, pc, 0);
        if (d.dx && !pl->pair) g[n++] = dx_gemm(p, *pl, pc, 0, 0);
        if (d.dw && !outer_dw(p, *pl)) g[n++] = dw_gemm(p, *pl, pc, 0);
        for (int i = 0; i < n; ++i) {
            size_t bytes = 0;
            if ((rc = losses_gemm_workspace(&g[i], pl->padded, &bytes))) return rc;
            pl->gemm_ws_bytes = std::max<uint64_t>(pl->gemm_ws_bytes, bytes);
        }
    }
    pl->gemm_ws = take(pl->gemm_ws_bytes);
    pl->bytes = at;
    return T0G_OK;
}

uint64_t weight_span(const t0g_linear_ce_desc &d) { return (uint64_t)(d.transpose == T0G_NT ? d.vocab : d.hidden) * d.ldw; }

// The GEMMs take operands of any size in whole 16-byte pieces and below 2^31 values otherwise.  A larger
// weight goes in pieces below that where a product would refuse the whole: narrower ones of rows of tokens,
// copies of a few tokens' columns.
int make_loss_plan(const Problem &p, Plan *pl) {
    int rc = plan_pieces(p, false, pl);
    if (rc == T0G_ERR_INVALID_ARG && weight_span(p.d) >= (1ull << 31)) {
        *pl = Plan();
        rc = plan_pieces(p, true, pl);
    }
    const uint64_t span = (uint64_t)p.d.rows * std::max(p.d.ldx, p.d.hidden);
    if (rc == T0G_ERR_INVALID_ARG && span >= (1ull << 31))
        return fail(rc, "x spans %llu elements: from 2^31 on the hidden size and the vocabulary must be multiples of 8",
                    (unsigned long long)span);
    return rc;
}

int run_gemm(t0g_device *dev, t0g_gemm_desc g, const Plan &pl, uint64_t base) {
    g.workspace = base + pl.gemm_ws;
    g.workspace_bytes = pl.gemm_ws_bytes;
    return losses_gemm(dev, &g, pl.padded);
}

// The copy of a piece of an unaligned weight.
int run_copy(t0g_device *dev, const Problem &p, const Plan &pl, const Piece &pc, uint64_t base) {
    const t0g_linear_ce_desc &d = p.d;
    T0gLossCopyArgs c;
    memset(&c, 0, sizeof c);
    c.src = weight_piece(p, d.w, pc.v0, d.ldw, 2);
    c.dst = base + pl.w;
    c.rows = d.transpose == T0G_NT ? pc.cols : d.hidden;
    c.cols = d.transpose == T0G_NT ? d.hidden : pc.cols;
    c.lds = d.ldw;
    c.ldd = ldw_of(p, pl, pc);
    const uint64_t groups = ((uint64_t)c.rows * (c.ldd / 8) + 255) / 256;
    return losses_launch(dev, "t0g_loss_copy_weight", (uint32_t)std::min<uint64_t>(groups, 1u << 20), 1, &c, sizeof c);
}

int run_dw(t0g_device *dev, const Problem &p, const Plan &pl, const Piece &pc, uint64_t base) {
    const t0g_linear_ce_desc &d = p.d;
    const t0g_gemm_desc g = dw_gemm(p, pl, pc, base);
    if (!outer_dw(p, pl)) return run_gemm(dev, g, pl, base);
    if (g.m == 0 || g.n == 0) return T0G_OK;
    T0gLossOuterArgs o;
    memset(&o, 0, sizeof o);
    o.a = g.a;
    o.b = g.b;
    o.c = g.c;
    o.rows = g.k;
    o.m = g.m;
    o.n = g.n;
    o.lda = g.lda;
    o.ldb = g.ldb;
    o.ldc = g.ldc;
    o.out_bf16 = g.out_dtype == T0G_BF16;
    o.vec = g.ldc % 8 == 0 && g.c % 16 == 0;
    o.stream = g.c % 128 == 0 && (uint64_t)g.ldc * dtype_size(g.out_dtype) % 128 == 0;
    o.m_inner = d.transpose == T0G_NN;   // the columns of x, which every block of G meets
    const uint64_t tiles = (((uint64_t)g.m + 31) / 32) * (((uint64_t)g.n + 127) / 128);
    const char *symbol = g.k <= 32 ? "t0g_loss_outer_1" : g.k <= 64 ? "t0g_loss_outer_2" : "t0g_loss_outer_4";
    return losses_launch(dev, symbol, (uint32_t)((tiles + 3) / 4), 1, &o, sizeof o);
}

// The whole rows' kernel for a vocabulary.
struct RowKernel {
    const char *symbol;
    uint32_t threads;
};
RowKernel row_kernel_for(uint32_t vocab) {
    if (vocab <= 256) return {"t0g_loss_row_1x1", 64};
    if (vocab <= 1024) return {"t0g_loss_row_1x4", 256};
    if (vocab <= 4096) return {"t0g_loss_row_4x4", 256};
    if (vocab <= 8192) return {"t0g_loss_row_8x4", 256};
    return {"t0g_loss_row_4x16", 1024};
}

// One of the 256x256 kernels on a piece: statistics, statistics with the exponentials kept, or G.
enum class Tile { Stats, Keep, Grad };
int run_tile(t0g_device *dev, Tile kind, const Problem &p, const Plan &pl, const Piece &pc, const T0gLossArgs &a,
             uint64_t base) {
    const t0g_linear_ce_desc &d = p.d;
    T0gLossGemmArgs t;
    memset(&t, 0, sizeof t);
    t.g.a = x_of(p, pl, base);
    t.g.b = w_of(p, pl, pc, base);
    t.g.c = p.grad ? base + pl.g : 0;
    t.g.m = d.rows;
    t.g.n = pc.cols;
    t.g.k = d.hidden;
    t.g.lda = ldx_of(p, pl);
    t.g.ldb = ldw_of(p, pl, pc);
    t.g.ldc = ld_of_g(pl, pc);
    t.g.tiles_m = round_up(d.rows, 256) / 256;
    t.g.tiles_n = round_up(pc.cols, 256) / 256;
    t.g.group_m = 8;
    t.g.flags = T0G_FLAG_XCD_REMAP;
    // the 256x256 GEMM kernels' rule for touching the lines of later stages
    const uint64_t wgs = (uint64_t)t.g.tiles_m * t.g.tiles_n;
    if (2.0 * d.hidden * ((double)d.rows + pc.cols) >= 96e6 &&
        (wgs <= 2 * kNumCUs || (t.g.tiles_m & (t.g.tiles_m - 1)) == 0))
        t.g.flags |= T0G_FLAG_PREFETCH;
    t.part = a.part + (uint64_t)pc.chunk0 * d.rows * 8;
    t.part2 = a.part2 ? a.part2 + (uint64_t)pc.chunk0 * d.rows * 4 : 0;
    t.ent_tok = a.ent_tok;
    t.ent_z = a.ent_z;
    t.ent_off = a.ent_off;
    t.row_par = a.row_par;
    t.v0 = pc.v0;
    t.slots = pl.slots;
    t.off_ld = pl.off_ld;
    t.flags = a.flags;
    t.k = a.k;
    t.r = a.r;
    static const char *symbols[3][2] = {{"t0g_loss_logits_nt", "t0g_loss_logits_nn"},
                                        {"t0g_loss_logits_nt_kept", "t0g_loss_logits_nn_kept"},
                                        {"t0g_loss_again_nt", "t0g_loss_again_nn"}};
    return losses_launch(dev, symbols[(int)kind][d.transpose == T0G_NN], (uint32_t)wgs, 1, &t, sizeof t);
}

int run_loss(t0g_device *dev, const Problem &p) {
    const t0g_linear_ce_desc &d = p.d;
    Plan pl;
    int rc = make_loss_plan(p, &pl);
    if (rc) return rc;
    uint64_t base = 0;
    if ((rc = losses_begin(dev, pl.bytes, &base))) return rc;
    if (d.rows == 0) {
        for (const Piece &pc : pl.pieces)   // a product over no rows: zeros
            if (d.dw && (rc = run_dw(dev, p, pl, pc, base))) return rc;
        return ok();
    }
    T0gLossArgs a;
    memset(&a, 0, sizeof a);
    a.x = d.x;
    a.xz = pl.copy_x || p.grad ? base + pl.xz : 0;
    a.labels = d.labels;
    a.dloss = d.dloss;
    a.loss = d.loss;
    a.lse = d.lse;
    a.ent_tok = base + pl.ent_tok;
    a.ent_q = base + pl.ent_q;
    a.ent_z = base + pl.ent_z;
    a.row_ent = base + pl.row_ent;
    a.row_sub = base + pl.row_sub;
    a.row_par = p.grad ? base + pl.row_par : 0;
    a.part = base + pl.part;
    a.part2 = p.dual ? base + pl.part2 : 0;
    a.z = base + pl.z;
    a.g = p.grad ? base + pl.g : 0;
    a.ent_off = pl.off_ld ? base + pl.ent_off : 0;
    a.off_ld = pl.off_ld;
    a.rows = d.rows;
    a.vocab = d.vocab;
    a.hidden = d.hidden;
    a.ldx = d.ldx;
    a.ldxz = pl.ldxz;
    a.slots = pl.slots;
    a.logit_scale = d.logit_scale;
    a.loss_scale = d.loss_scale;
    a.tau = 1.0f;
    a.label_weight = 1.0f;
    if (d.label_type == T0G_I64) a.flags |= T0G_LOSS_LABEL64;
    if ((d.x & 15) == 0 && d.ldx % 8 == 0 && d.hidden % 8 == 0) a.flags |= T0G_LOSS_X_VEC;
    if (p.t) {
        a.teacher = p.t->teacher;
        a.tokens = p.t->tokens;
        a.top_k = p.t->top_k;
        a.ldt = p.ldt;
        a.tau = p.t->temperature;
        a.label_weight = p.t->label_weight;
        a.distill_weight = p.t->distill_weight;
        if (p.t->token_type == T0G_I64) a.flags |= T0G_LOSS_TOKEN64;
        if (p.t->teacher_dtype == T0G_BF16) a.flags |= T0G_LOSS_TEACHER16;
    }
    if (p.dual) a.flags |= T0G_LOSS_DUAL;
    if (pl.direct) a.flags |= T0G_LOSS_DIRECT;
    if (pl.pair) a.flags |= T0G_LOSS_PAIR;
    if (!pl.fused && pl.pieces.size() == 1) a.flags |= T0G_LOSS_Z;
    a.chunks = pl.chunks;
    // with both softmaxes the first is the labels', else the only one
    const double k = (double)d.logit_scale * 1.4426950408889634;
    a.k = (float)(p.dual || !p.t ? k : k / p.t->temperature);
    a.r = p.dual ? 1.0f / p.t->temperature : 1.0f;

    auto row_kernel = [&](const char *symbol, uint32_t rows_per_group) {
        const uint32_t groups = (uint32_t)(((uint64_t)d.rows + rows_per_group - 1) / rows_per_group);
        return losses_launch(dev, symbol, std::min<uint32_t>(groups, 1u << 20), 1, &a, sizeof a);
    };
    auto at_piece = [&](const Piece &pc) {
        a.v0 = pc.v0;
        a.cols = pc.cols;
        a.ldz = round_up(pc.cols, 4);
        a.ldg = ld_of_g(pl, pc);
        a.chunk0 = pc.chunk0;
    };
    auto piece_kernel = [&](const char *symbol, uint32_t groups) {
        return losses_launch(dev, symbol, groups, std::min(d.rows, kMaxGridY), &a, sizeof a);
    };
    const size_t n = pl.pieces.size();
    // by rows: one kernel for all of a row that fits a workgroup's registers
    const bool one = !pl.fused && n == 1 && d.vocab <= T0G_LOSS_ROW_MAX;
    auto whole_rows = [&] {
        const RowKernel k = row_kernel_for(d.vocab);
        return losses_launch(dev, k.symbol, std::min<uint32_t>(d.rows, 1u << 20), 1, &a, sizeof a, k.threads);
    };
    if (!pl.direct) {
        // a wave takes a row of fewer than 64 entries
        const bool wave = pl.slots < 64;
        if ((rc = wave ? row_kernel("t0g_loss_prepare", 4) : row_kernel("t0g_loss_prepare_long", 1))) return rc;
    }
    for (size_t i = 0; i < n; ++i) {
        const Piece &pc = pl.pieces[i];
        at_piece(pc);
        if (pl.copy_w && (rc = run_copy(dev, p, pl, pc, base))) return rc;
        if (pl.fused)
            rc = run_tile(dev, pl.keep && i + 1 == n ? Tile::Keep : Tile::Stats, p, pl, pc, a, base);
        else if (!(rc = run_gemm(dev, logits_gemm(p, pl, pc, base), pl, base)) && !one)
            rc = piece_kernel("t0g_loss_stats", pc.chunks);
        if (rc) return rc;
    }
    if (pl.fused || (!p.grad && !one)) {
        // 16 rows read a chunk's statistics as one line; fewer where that leaves CUs idle
        while (a.row_shift < 4 && d.rows >> (a.row_shift + 1) >= 2 * kNumCUs) ++a.row_shift;
        if ((rc = row_kernel("t0g_loss_combine", 1u << a.row_shift))) return rc;
    } else if (!p.grad) {
        if ((rc = whole_rows())) return rc;
    }
    if (!p.grad) return ok();

    T0gLossSumArgs s;
    memset(&s, 0, sizeof s);
    s.planes = base + pl.planes;
    s.rows = d.rows;
    s.cols = d.hidden;
    s.ldp = pl.ldp;
    // few rows: dx reads the weight again while the caches may hold it, before dW is written (100 rows of
    // 32000x1024: 96.1 us against 94.5; with the GEMM's dW and 64 rows of 128000x4096 804 against 846)
    const bool dx_first = pl.pair && d.dx && (outer_dw(p, pl) || (uint64_t)d.vocab * d.hidden * 2 <= kCacheBytes);
    uint32_t planes = 0;
    for (size_t i = n; i-- > 0;) {
        const Piece &pc = pl.pieces[i];
        at_piece(pc);
        if (pl.copy_w && i + 1 < n && (rc = run_copy(dev, p, pl, pc, base))) return rc;
        if (pl.keep && i + 1 == n) {
            rc = piece_kernel("t0g_loss_grad_kept", (a.ldg + 2047) / 2048);
        } else if (pl.fused) {
            if (!(rc = run_tile(dev, Tile::Grad, p, pl, pc, a, base))) rc = row_kernel("t0g_loss_grad_entries", 4);
        } else if (one) {
            rc = whole_rows();
        } else {
            if (i + 1 == n || !(rc = run_gemm(dev, logits_gemm(p, pl, pc, base), pl, base)))
                rc = piece_kernel("t0g_loss_grad", (pc.cols + T0G_LOSS_CHUNK - 1) / T0G_LOSS_CHUNK);
        }
        if (rc || (d.dw && !dx_first && (rc = run_dw(dev, p, pl, pc, base)))) return rc;
        if (!d.dx) continue;
        const t0g_gemm_desc dx = dx_gemm(p, pl, pc, base, planes);
        uint32_t splits = 1;
        if (pl.pair) {
            if ((rc = losses_gemm_planes_count(&dx, pl.padded, &splits)) || (rc = losses_gemm_planes(dev, &dx, pl.padded)))
                return rc;
            if (d.dw && dx_first && (rc = run_dw(dev, p, pl, pc, base))) return rc;
        } else if ((rc = run_gemm(dev, dx, pl, base))) {
            return rc;
        }
        if (pl.group == 0) continue;
        if (++planes < pl.group && i > 0) continue;
        // the planes so far, onto those before
        const bool last = i == 0;
        s.n = pl.pair ? 2 * splits : planes;
        s.out = last ? d.dx : base + pl.acc;
        s.ldo = last ? d.lddx : pl.ldp;
        s.out_bf16 = last && d.dx_dtype == T0G_BF16;
        s.vec = d.hidden % 4 == 0 && s.ldo % 4 == 0 && s.out % 16 == 0;
        const uint64_t items = (uint64_t)d.rows * (d.hidden / (s.vec ? 4 : 1));
        const uint32_t groups = (uint32_t)std::min<uint64_t>((items + 255) / 256, 1u << 16);
        if ((rc = losses_launch(dev, "t0g_loss_sum", groups, 1, &s, sizeof s))) return rc;
        s.acc = base + pl.acc;
        planes = 0;
    }
    return ok();
}

// No exception leaves a C entry: a vocabulary in very many pieces has a long list of them.
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::exception &e) {
        return fail(T0G_ERR_OUT_OF_MEMORY, "host: %s", e.what());
    }
}

int loss_call(t0g_device *dev, const t0g_linear_ce_desc *d, const t0g_linear_distill_desc *t) {
    return guarded([&] {
        if (!dev) return fail(T0G_ERR_INVALID_ARG, "device is NULL");
        if (!d) return fail(T0G_ERR_INVALID_ARG, "desc is NULL");
        Problem p;
        int rc = check_problem(d, t, &p);
        if (rc) return rc;
        std::lock_guard<std::mutex> lk(device_mutex(dev));
        return run_loss(dev, p);
    });
}

int loss_scratch(const t0g_linear_ce_desc *d, const t0g_linear_distill_desc *t, size_t *bytes) {
    return guarded([&] {
        if (!d || !bytes) return fail(T0G_ERR_INVALID_ARG, "NULL argument");
        *bytes = 0;
        Problem p;
        Plan pl;
        int rc = check_problem(d, t, &p);
        if (rc || (rc = make_loss_plan(p, &pl))) return rc;
        *bytes = pl.bytes;
        return ok();
    });
}

}  // namespace
}  // namespace t0g

extern "C" {

int t0g_linear_cross_entropy(t0g_device *dev, const t0g_linear_ce_desc *desc) {
    return t0g::loss_call(dev, desc, nullptr);
}

int t0g_linear_distill(t0g_device *dev, const t0g_linear_distill_desc *desc) {
    return t0g::loss_call(dev, desc ? &desc->head : nullptr, desc);
}

int t0g_set_loss_form(uint32_t form) {
    if (form > T0G_LOSS_FORM_FUSED) return t0g::fail(T0G_ERR_INVALID_ARG, "loss form %u", form);
    t0g::g_form.store(form);
    return t0g::ok();
}

int t0g_linear_cross_entropy_scratch_size(const t0g_linear_ce_desc *desc, size_t *bytes) {
    return t0g::loss_scratch(desc, nullptr, bytes);
}

int t0g_linear_distill_scratch_size(const t0g_linear_distill_desc *desc, size_t *bytes) {
    return t0g::loss_scratch(desc ? &desc->head : nullptr, desc, bytes);
}

}  // extern "C"
