// attend.hip - the plan of an attention call over two ranges of keys: which
// kernel shapes of attend.hpp, how the key tiles are cut into runs, where
// partial results wait.
#include <math.h>

#include "internal.hpp"

namespace aotk {

template <int KIND>
void att_launch_kind(int head_dim, int p, int o, const AttendLaunch &a, uint32_t blocks, hipStream_t s);
template <int KIND>
void att_join_kind(int head_dim, const AttendLaunch &a, uint32_t prefix_chunks, uint32_t total, uint32_t first_row, uint64_t items, uint32_t runs, hipStream_t s);

// Rows of a shape's tile, and keys.
static int att_rows(int shape) { return shape <= 2 ? 16 * shape : (shape == 3 ? 64 : 128); }
static int att_keys(int kind, int head_dim, int shape) {
    if (shape <= 2) return kind == AOTK_F32 ? 16 : 32;
    return kind == AOTK_F32 || head_dim == 256 ? 32 : 64;
}

struct AttPart {
    int shape;
    int rows_tile, nk;
    uint32_t run;  // key tiles of a block
};

static uint32_t att_row_tiles(uint32_t rows, uint32_t group, int rows_tile) {
    return (uint32_t)(((uint64_t)rows * group + rows_tile - 1) / rows_tile);
}

// Key tiles of a sequence's row tile.
static uint64_t att_tiles(const AttendArgs &a, uint64_t na, bool causal, const AttendSeq &s, uint32_t group, const AttPart &p, uint32_t tile) {
    const uint64_t all = (uint64_t)s.rows * group, r0 = (uint64_t)tile * p.rows_tile;
    const uint64_t r1 = r0 + p.rows_tile < all ? r0 + p.rows_tile : all;
    const int64_t first = (int64_t)s.len - s.rows;
    const int64_t pmin = causal ? first + (int64_t)(r0 / group) : (int64_t)s.len - 1;
    const int64_t pmax = causal ? first + (int64_t)((r1 - 1) / group) : (int64_t)s.len - 1;
    const AttendSpan sp = attend_span(na, causal ? a.window : 0, causal ? a.n_sink : 0, pmin, pmax);
    return (sp.na + p.nk - 1) / p.nk + (sp.nb + p.nk - 1) / p.nk;
}

// The runs of one range's blocks (the prefix's or the sequences' own).
static void att_cut(int kind, int head_dim, const AttendArgs &a, uint64_t na, bool causal, const AttendSeq *seqs, size_t n, uint32_t group, AttPart &p) {
    p.rows_tile = att_rows(p.shape);
    p.nk = att_keys(kind, head_dim, p.shape);
    uint64_t tiles = 0, items = 0;
    for (size_t i = 0; i < n; i++) {
        if (!seqs[i].rows) continue;
        const uint32_t rt = att_row_tiles(seqs[i].rows, group, p.rows_tile);
        items += rt;
        tiles += att_tiles(a, na, causal, seqs[i], group, p, rt - 1) * rt;
    }
    p.run = 1;
    if (!items || !tiles) return;
    tiles *= a.n_kv_head;
    items *= a.n_kv_head;
    // As many runs as fill the chip (512 blocks are resident at two a CU), unless
    // writing and joining their results (f32, for every row) would cost more than
    // the tiles of a run: c runs of T tiles take T / c tile times and c times the
    // traffic of one result. Measured around that optimum (times 0.7 / 1 / 1.5 of
    // its c): 64 sequences behind 8192 bf16, weights rounded, 56 / 52 / 57 us, 64 f32
    // rows in a 1024 window 53 / 47 / 54 us. Few rows: runs of one tile a wave at least (of two: 27
    // -> 30 us for a 1024 window, one f32 row).
    const bool narrow = p.shape <= 2;
    const double want = 512, least = narrow ? 4 : 1;
    const double each = (double)tiles / (double)items;  // of a row tile, on average
    double run;
    if ((double)items >= want) {
        run = (double)tiles / want + 3;  // whole row tiles, but for those far longer than the others
    } else {
        double cuts = want / (double)items;
        if (!narrow) {
            // what a CU reaches; heads of 256 leave one wave a SIMD
            const double rate = kind == AOTK_F32 ? 0.5e6 : (head_dim == 256 ? 2.0e6 : 3.5e6);
            const double tile_us = 4.0 * p.rows_tile * p.nk * head_dim / rate;
            const double part_us = (double)items * p.rows_tile * head_dim * 8 / 4e6;
            const double most_cuts = sqrt(each * tile_us / part_us);
            cuts = cuts < most_cuts ? cuts : most_cuts;
        }
        run = ceil(each / floor(cuts < 1 ? 1 : cuts));
    }
    run = run > least ? run : least;
    p.run = run < 0x7fffffff ? (uint32_t)run : 0x7fffffffu;
}

static uint32_t att_chunks(const AttendArgs &a, uint64_t na, bool causal, const AttendSeq &s, uint32_t group, const AttPart &p) {
    if (!s.rows) return 0;
    const uint32_t rt = att_row_tiles(s.rows, group, p.rows_tile);
    // spans grow with the position until the window is full: the last tile's is the longest, or within a tile of it
    uint64_t t = att_tiles(a, na, causal, s, group, p, rt - 1);
    if (causal && rt > 1) {
        const uint64_t u = att_tiles(a, na, causal, s, group, p, rt - 2);
        t = t > u ? t : u;
        t += 2;
    }
    const uint64_t c = (t + p.run - 1) / p.run;
    return (uint32_t)(c ? c : 1);
}

// The shape for that many rows (x group) of one sequence, or of all.
static int att_shape(uint64_t rows, int head_dim) {
    if (rows <= 16) return 1;
    if (rows <= 32 && head_dim < 256) return 2;
    return rows <= 64 ? 3 : 4;
}

struct AttWhole {
    AttPart prefix, own;
    bool grouped;            // the prefix has blocks of its own, over all sequences' rows
    uint32_t prefix_chunks, total, group;
    uint64_t slots;          // partial results, in rows
    bool any_parts;
};

static AttWhole att_whole(int kind, int head_dim, const AttendArgs &a, const AttendSeq *seqs, size_t n) {
    AttWhole w = {};
    w.group = a.n_head / a.n_kv_head;
    uint64_t total = 0, most = 0, with_rows = 0, own_tiles = 0;
    for (size_t i = 0; i < n; i++) {
        total += seqs[i].rows;
        own_tiles += att_row_tiles(seqs[i].rows, w.group, 128);
        most = most > seqs[i].rows ? most : seqs[i].rows;
        with_rows += seqs[i].rows > 0;
    }
    w.total = (uint32_t)total;
    // Beyond 1024 tiles of 16-bit rows, each sequence's blocks read the prefix for
    // themselves: the products bound them, and results of two parts for every row
    // need not be joined (bf16, 32 heads over 4 of 64: 16 sequences of 512 rows behind
    // 4096 323 -> 261 us, 16 of 1024 behind 512 277 -> 151). With fewer, and with f32
    // (32 over 8 of 128: 8 of 1024 behind 4096 2403 -> 2863 us), sharing is faster.
    // Sequences of few rows among them would waste tiles: a quarter at most.
    const uint64_t packed = att_row_tiles((uint32_t)total, w.group, 128);
    const bool alone = kind != AOTK_F32 && packed * a.n_kv_head >= 1024 && own_tiles * 4 <= packed * 5;
    w.grouped = a.n_prefix > 0 && with_rows > 1 && !alone;
    w.own.shape = att_shape(most * w.group, head_dim);
    if (w.grouped) {
        w.prefix.shape = att_shape(total * w.group, head_dim);
        // pairs that have a kernel: the same shape, or few rows beside many (32 beside
        // 64 for 16 bits only, where the own range's shape decides how weights are
        // rounded; for f32 64 beside 64: 3 sequences of 20 heads behind 4096 33.3 -> 32.8 us)
        if (w.prefix.shape == 2 || (w.prefix.shape == 3 && w.own.shape == 2 && kind == AOTK_F32) || w.own.shape >= 3)
            w.own.shape = w.prefix.shape;
        const AttendSeq all = {0, w.total, a.n_prefix, 0};
        att_cut(kind, head_dim, a, 0, false, &all, 1, w.group, w.prefix);
        w.prefix_chunks = att_chunks(a, 0, false, all, w.group, w.prefix);
        w.slots = (uint64_t)w.prefix_chunks * total;
        w.any_parts = true;
    } else {
        w.prefix.shape = w.own.shape;
    }
    const uint64_t na = w.grouped ? 0 : a.n_prefix;
    att_cut(kind, head_dim, a, na, true, seqs, n, w.group, w.own);
    for (size_t i = 0; i < n; i++) {
        const uint32_t c = att_chunks(a, na, true, seqs[i], w.group, w.own);
        if (c > 1 || w.grouped) {
            w.slots += (uint64_t)c * seqs[i].rows;
            w.any_parts = true;
        }
    }
    return w;
}

size_t attend_scratch_bytes(int kind, int head_dim, const AttendArgs &a, const AttendSeq *seqs, size_t n) {
    const AttWhole w = att_whole(kind, head_dim, a, seqs, n);
    return w.any_parts ? align_up(w.slots * a.n_head * 8, 256) + w.slots * a.n_head * head_dim * 4 : 0;
}

void launch_attend(int kind, int head_dim, const AttendArgs &a, const AttendSeq *seqs, size_t n, void *scratch, hipStream_t s) {
    const AttWhole w = att_whole(kind, head_dim, a, seqs, n);
    AttendLaunch l = {};
    l.q = a.q;
    l.out = a.out;
    l.n_head = a.n_head;
    l.n_kv_head = a.n_kv_head;
    l.scale_log2 = a.scale * 1.44269504088896340736f;
    if (w.any_parts) {
        l.part_ml = (float *)scratch;
        l.part_acc = (float *)((uint8_t *)scratch + align_up(w.slots * a.n_head * 8, 256));
    }
    l.joined = w.grouped;
    AttendView &own = l.range[0], &pre = l.range[1];
    own.k = own.ka = a.k;
    own.v = own.va = a.v;
    own.window = a.window;
    own.n_sink = a.n_sink;
    own.run = w.own.run;
    own.causal = 1;
    if (w.grouped) {
        l.seq[ATTEND_SEQS] = {0, w.total, a.n_prefix, 0, 0, w.prefix_chunks, 0};
        l.prefix_blocks = att_row_tiles(w.total, w.group, w.prefix.rows_tile) * w.prefix_chunks * a.n_kv_head;
        pre.k = pre.ka = a.k_prefix;
        pre.v = pre.va = a.v_prefix;
        pre.run = w.prefix.run;
        pre.seq0 = ATTEND_SEQS;
    } else if (a.n_prefix) {
        own.ka = a.k_prefix;
        own.va = a.v_prefix;
        own.na = a.n_prefix;
    }
    uint64_t part = (uint64_t)w.prefix_chunks * w.total;
    for (size_t b0 = 0; b0 < n;) {
        uint32_t blocks = 0, first_row = 0, last_row = 0, runs = 0;
        bool parts = false;
        l.n_seq = 0;
        for (; b0 < n && l.n_seq < ATTEND_SEQS; b0++) {
            const AttendSeq &q = seqs[b0];
            if (!q.rows) continue;
            const uint32_t c = att_chunks(a, own.na, true, q, w.group, w.own);
            if (l.n_seq == 0) first_row = q.row0;
            last_row = q.row0 + q.rows;
            l.seq[l.n_seq++] = {q.row0, q.rows, q.len, q.cache, blocks, c, part};
            if (c > 1 || w.grouped) {
                part += (uint64_t)c * q.rows;
                parts = true;
                runs = runs > c + w.prefix_chunks ? runs : c + w.prefix_chunks;
            }
            blocks += att_row_tiles(q.rows, w.group, w.own.rows_tile) * c * a.n_kv_head;
        }
        if (!l.n_seq) continue;
        blocks += l.prefix_blocks;
        own.block0 = l.prefix_blocks;
        (kind == AOTK_F32   ? att_launch_kind<AOTK_F32>
         : kind == AOTK_F16 ? att_launch_kind<AOTK_F16>
                            : att_launch_kind<AOTK_BF16>)(head_dim, w.prefix.shape, w.own.shape, l, blocks, s);
        l.prefix_blocks = 0;  // done with the first sequences
        // (a launch holds less than 2^32 threads)
        const uint32_t most = (1u << 21) / a.n_head / 4 * 4;
        for (uint32_t r = first_row; parts && r < last_row; r += most) {
            const uint32_t rows = last_row - r < most ? last_row - r : most;
            (kind == AOTK_F32   ? att_join_kind<AOTK_F32>
             : kind == AOTK_F16 ? att_join_kind<AOTK_F16>
                                : att_join_kind<AOTK_BF16>)(head_dim, l, w.prefix_chunks, w.total, r, (uint64_t)rows * a.n_head, runs, s);
        }
    }
}

}  // namespace aotk
