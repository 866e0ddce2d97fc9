// How the training operators are cut, on the host and without a GPU: tiles and splits of products, elementwise passes, workspaces
// (linear.hip, pack8.hip).
#pragma once
#include "pifu_internal.h"

static inline int pifu_elem_bytes(int dtype) { return dtype == PIFU_F32 ? 4 : 2; }

// How an elementwise pass over a matrix is cut: a block of 256 lanes takes tx * 8 columns (64 lanes' worth, more where there are fewer
// rows than lanes for them) and 256 / tx rows at a time, four times over at once, so that a lane has the loads of four rows in flight.
// Every block has a range of rows to itself.  About 8 blocks per CU, `most` blocks of rows at most.
struct RowCut {
    int64_t blocks = 1, rows = 1, wide = 1;
    int tx = 1;
    RowCut() = default;
    RowCut(int64_t m, int64_t cols, int64_t most)
    {
        while (tx * 8 < cols && (tx < 64 || (tx < 256 && 256 / tx > m))) tx *= 2;
        wide = (cols + tx * 8 - 1) / (tx * 8);
        const int64_t group = 4 * (256 / tx), groups = m > 0 ? (m + group - 1) / group : 1;
        blocks = 2048 / wide;
        if (blocks > most) blocks = most;
        if (blocks < 1) blocks = 1;
        rows = (groups + blocks - 1) / blocks * group;
        blocks = (groups * group + rows - 1) / rows;
    }
};

constexpr unsigned DMA_SPAN = 0x7fffffffu;       // bytes one tile of a DMA operand may span (32-bit offsets), and the zero offset's start
constexpr int FEW_ROWS = PIFU_LINEAR_FEW_ROWS;   // rows of a forward pass without matrix instructions
constexpr int NARROW = 4;                        // outputs of a backward pass without matrix instructions
constexpr int64_t MAX_BLOCKS = 0xffffffffll / 256;       // blocks of 256 lanes in a launch: 2^32 - 1 lanes along x
constexpr int64_t MAX_WIDTH = 65535 * 256;         // n and k: 256 columns per block of a grid whose y extent is 65535 at most

// Whether an operand can go by LDS-DMA: whole 16-byte chunks at 16-byte addresses, and 32-bit offsets inside a tile of up to 256 rows
// (rows of less than 8 MiB).  That holds for the library's own copies too, whose addresses are aligned and whose rows are whole chunks.
inline bool dma_pitch_ok(int elem, int64_t ld) { return ld * elem % 16 == 0 && ld * elem < (int64_t)DMA_SPAN / 256; }
inline bool dma_ok(int elem, const void *x, int64_t ld, int64_t cols)
{
    return (uintptr_t)x % 16 == 0 && dma_pitch_ok(elem, ld) && cols * elem % 16 == 0;
}

// How a product is cut: tile size, and the split of the tiles that do not fill a last round of the chip's 256 CUs.  tiles_i = 0: more
// tiles than a launch holds, whatever their size.
struct Cut {
    int tile = 0;                      // 0: 64 x 64, 1: 128 x 128, 2: 256 x 256
    bool a_dma = false, b_dma = false; // whether the operands come by LDS-DMA: both do where the tile is 256 x 256
    int64_t tiles_i = 0, tiles_j = 0, whole = 0, splits = 1, per = 0;
    int64_t rest() const { return tiles_i * tiles_j - whole; }
    int64_t bytes() const { const int64_t b = 64 << tile; return splits > 1 ? rest() * splits * b * b * 4 : 0; }
};

// The cut with the least predicted time.  A CU is taken to work on `slots` blocks at a time (LDS holds 5, 2 and 1; the fit has 4 for the
// smallest); a p tile of a block takes `work` cycles of the CU's matrix pipes, or `alone` cycles where too few blocks share the CU to
// hide the transfers; a tile costs `ends` for its first transfers and its epilogue, and parts cost their way through memory and one more
// launch.  Fitted to a sweep over tile sizes and splits of 23 products from 16 MFLOP to 84 GFLOP (profiles/training_products_sweep.txt):
// of the 19 whose choice was timed there, it takes 1.04 times the best one's time in the mean, 1.13 at worst.
// `runs`: how often the sum over p is run through (operands in halves; not on the largest tile).
inline Cut plan_product(int elem, int64_t I, int64_t J, int64_t P, bool a_dma, bool b_dma, int runs = 1)
{
    const bool dma = a_dma && b_dma;
    static const int slots[3] = {4, 2, 1};
    static const double work16[3] = {480, 1250, 3300}, alone16[3] = {1200, 1650, 3300}, work32[2] = {1400, 4700}, alone32[2] = {2600, 6500};
    static const double ends[3] = {3500, 6000, 24000};
    constexpr int64_t CUS = 256;
    Cut best;
    double best_time = 0;
    const int64_t bk = 128 / elem, depth = (P + bk - 1) / bk * runs;
    for (int tile = 0; tile < (elem == 2 && dma && runs == 1 ? 3 : 2); tile++) {
        const double work = elem == 2 ? work16[tile] : work32[tile];
        const double alone = (elem == 2 ? alone16[tile] : alone32[tile]) * (dma ? 1 : 1.3);        // (fetched through registers)
        const int64_t b = 64 << tile;
        Cut c;
        c.tile = tile;
        c.a_dma = a_dma;
        c.b_dma = b_dma;
        c.tiles_i = (I + b - 1) / b;
        c.tiles_j = (J + b - 1) / b;
        if (c.tiles_i > (MAX_BLOCKS - 4096) / c.tiles_j) continue;   // (4096: the blocks of split tiles beside the whole ones)
        auto run = [&](int64_t blocks, int64_t deep) {
            const int64_t full = blocks / (CUS * slots[tile]), rest = (blocks - full * CUS * slots[tile] + CUS - 1) / CUS;
            auto round = [&](int64_t r) { return deep * (r * work > alone ? r * work : alone) + ends[tile]; };
            return full * round(slots[tile]) + (rest ? round(rest) : 0.0);
        };
        const int64_t tiles = c.tiles_i * c.tiles_j;
        for (int all = 0; all < 2; all++) {                          // split all tiles, or those behind the full rounds
            const int64_t whole = all ? 0 : tiles / CUS * CUS, rest = tiles - whole;
            if (all && tiles < CUS) break;
            for (int64_t s = 1; s <= depth || s == 1; s = s < 4 ? s + 1 : s + s / 4) {
                c.per = depth > 0 ? (depth + s - 1) / s : 0;
                c.splits = depth > 0 ? (depth + c.per - 1) / c.per : 1;
                c.whole = c.splits > 1 ? whole : tiles;
                double time = run(c.whole, depth);
                if (c.splits > 1) time += run(rest * c.splits, c.per) + 12000 + (double)c.bytes() * 2 / 3000;
                if (best_time == 0 || time < best_time) { best = c; best_time = time; }
                if (!rest || rest * s > 8 * CUS) break;              // (at most 4096 blocks with s > 1: s at most doubles)
            }
        }
    }
    return best;
}

struct Plan {
    int64_t dz = 0, h = 0, sums = 0, part = 0, total = 0;          // workspace: offsets, bytes
    bool scaled = false;               // gw from scaled fp16 operands
    bool halves_dz = false, halves_h = false;      // dz, h in halves: the second lies lddz, ldh columns behind the first
    int64_t dz16 = 0, exp_i = 0, exp_j = 0, max_i = 0, max_j = 0;
    RowCut max_cut_i, max_cut_j;       // the passes that look for the largest magnitudes of dz and h
    Cut gx, gw;
    int64_t lddz = 0, ldh = 0;         // whole chunks of a row of dz, h
    int64_t pitch_dz() const { return lddz * (halves_dz ? 2 : 1); }
    int64_t pitch_h() const { return ldh * (halves_h ? 2 : 1); }
    RowCut cut;
    bool narrow = false, fits = true;  // fits: one launch holds each product
    int64_t w = 0, ldw = 0;            // w with rows that the product can fetch by LDS-DMA
};

// Whether a copy of an operand with 16-byte aligned rows of `pitch` elements pays: each of its elements enters `times` products, of
// `size` in all.  Without LDS-DMA a product is fetched through registers and held to smaller tiles.
inline bool copy_pays(int elem, int64_t pitch, int64_t times, int64_t size)
{
    return times >= 512 && size >= (int64_t)1 << 31 && dma_pitch_ok(elem, pitch);
}

inline bool decodes(const pifu_linear_grad_args &g)
{
    const int elem = pifu_elem_bytes(g.dtype);
    return g.gw && (!g.x || g.x_act != PIFU_ACT_NONE ||
                    (!dma_ok(elem, g.x, g.ldx, g.k) && copy_pays(elem, round_up(g.k, 8), g.n, g.m * g.n * g.k)));
}

inline bool smooth(int act) { return act >= PIFU_ACT_SIGMOID; }

// Calls of up to this many multiplications a product take 16-bit operands that were computed on the way in as two halves, which keep
// their result at its own rounding; in larger ones, bound by the matrix instructions, they are rounded once (the result is off by 1.4
// times its own rounding) or scaled.  Backward pass with gelu, bf16, in us with halves / rounded once: 1000 x 128 x 256 26 / 21,
// 5000 x 512 x 1024 72 / 53, 50000 x 512 x 1024 372 / 240, 16384 x 4096 x 4096 2426 / 1035.  With gelu on both sides, halves / scaled:
// 5000 x 256 x 512 55 / 61, 5000 x 512 x 1024 86 / 82, 50000 x 512 x 1024 499 / 385.
constexpr int64_t HALVES_MOST = (int64_t)1 << 32;

constexpr int64_t MAX_PARTS = 128;     // blocks of rows of a column maximum

inline Plan plan_backward(const pifu_linear_grad_args &g)
{
    Plan p;
    int64_t at = 0;
    const int64_t e = pifu_elem_bytes(g.dtype);
    auto take = [&](int64_t bytes) { const int64_t from = at; at += round_up(bytes, 256); return from; };
    if (g.n <= NARROW && g.m > 0) {
        p.narrow = true;
        p.cut = RowCut(g.m, g.k, 512);
        p.total = g.gw || g.gb ? p.cut.blocks * ((g.gw ? g.n * g.k : 0) + g.n) * 4 : 0;
        return p;
    }
    const bool halves = e == 2 && g.m > 0 && g.m * g.n * g.k <= HALVES_MOST && dma_pitch_ok(2, 2 * round_up(g.n, 8)) &&
                        dma_pitch_ok(2, 2 * round_up(g.k, 8));           // (the halves come by LDS-DMA only)
    p.halves_dz = halves && smooth(g.act);
    p.halves_h = halves && smooth(g.x_act);
    // (scaled operands come by LDS-DMA only: rows too long for it stay in bf16)
    p.scaled = g.dtype == PIFU_BF16 && g.gw && g.m > 0 && smooth(g.act) && smooth(g.x_act) && !halves &&
               dma_pitch_ok(2, round_up(g.n, 8)) && dma_pitch_ok(2, round_up(g.k, 8));
    if (g.act != PIFU_ACT_NONE && (g.gx || g.gw)) p.lddz = round_up(g.n, 8);
    if (p.lddz && (g.gx || !p.scaled)) p.dz = take(g.m * p.pitch_dz() * e);
    if (p.scaled) {
        p.dz16 = take(g.m * p.lddz * 2);
        p.exp_i = take(g.n * 4);
        p.exp_j = take(g.k * 4);
        p.max_cut_i = RowCut(g.m, g.n, MAX_PARTS);
        p.max_cut_j = RowCut(g.m, g.k, MAX_PARTS);
        p.max_i = take(p.max_cut_i.blocks * g.n * 4);
        p.max_j = take(p.max_cut_j.blocks * g.k * 4);
    }
    if (decodes(g)) { p.ldh = round_up(g.k, 8); p.h = take(g.m * p.pitch_h() * e); }
    p.cut = RowCut(g.m, g.n, 256);
    if (g.gb) { p.sums = at; at += round_up(p.cut.blocks * g.n * 4, 256); }
    // the parts of gx and gw follow each other on the stream: one area
    const int elem = (int)e;
    const bool da = p.lddz ? dma_pitch_ok(elem, p.pitch_dz()) : dma_ok(elem, g.grad, g.ldg, g.n);
    int64_t part = 0;
    if (g.gx && g.m > 0) {
        const bool db = dma_ok(elem, g.w, g.ldw, g.k);
        const int runs = 1 + p.halves_dz;
        if (!db && copy_pays(elem, round_up(g.k, 8), runs * g.m, runs * g.m * g.n * g.k)) {
            p.ldw = round_up(g.k, 8);
            p.w = take(g.n * p.ldw * e);
        }
        p.gx = plan_product(elem, g.m, g.k, g.n, da, db || p.ldw, runs);
        part = p.gx.bytes();
        p.fits = p.gx.tiles_i > 0;
    }
    if (g.gw) {
        const bool db = p.ldh ? dma_pitch_ok(elem, p.pitch_h()) : dma_ok(elem, g.x, g.ldx, g.k);
        p.gw = plan_product(elem, g.n, g.k, g.m, da, db, 1 + p.halves_dz + p.halves_h);
        if (p.gw.bytes() > part) part = p.gw.bytes();
        p.fits = p.fits && p.gw.tiles_i > 0;
    }
    p.part = at;
    p.total = at + part;
    return p;
}

struct Forward {
    Cut cut;
    bool fits = true;                  // one launch holds the product
    int64_t ldx = 0, ldw = 0, x = 0, w = 0, total = 0;       // pitches of the copies of x and w (0: used where they lie), workspace offsets
};

inline Forward plan_forward(const pifu_linear_args &g)
{
    const int elem = pifu_elem_bytes(g.dtype);
    Forward f;
    if (g.m <= FEW_ROWS) return f;
    const bool da = dma_ok(elem, g.x, g.ldx, g.k), db = dma_ok(elem, g.w, g.ldw, g.k);
    const int64_t size = g.m * g.n * g.k, pitch = round_up(g.k, 8);
    if (!da && copy_pays(elem, pitch, g.n, size)) { f.ldx = pitch; f.x = f.total; f.total += round_up(g.m * pitch * elem, 256); }
    if (!db && copy_pays(elem, pitch, g.m, size)) { f.ldw = pitch; f.w = f.total; f.total += round_up(g.n * pitch * elem, 256); }
    f.cut = plan_product(elem, g.m, g.n, g.k, da || f.ldx, db || f.ldw);
    f.fits = f.cut.tiles_i > 0;
    f.total += f.cut.bytes();
    return f;
}
