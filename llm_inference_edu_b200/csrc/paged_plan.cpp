// Host side of the paged cache operators: admission of one step's batch and
// the work lists of its attention.  No device work.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <queue>
#include <vector>

#include "paged.cuh"

namespace qb {
namespace paged {
namespace {

// A row block before its units are cut.
struct Block {
    int32_t seq, kvh, row0, rows, ns, u0, units, w0, hi;
};

// How one kernel's blocks are cut.  Costs count in units of keys.
struct Grid {
    int unit;       // keys a unit
    int block;      // packed rows a block
    int slots;      // CTAs resident at once
    int fixed;      // cost of starting an item
    int part;       // further cost of an item that leaves a partial result
    int least;      // fewest units worth an item of its own
    int narrow, wide;  // a unit of a block of more than `narrow` rows costs `wide`
};

// The plain form of every variant: 8 rows and 64 keys a unit, one warp a row.
Grid rows_grid() { return Grid{64, 8, 148 * 4, 1, 1, 2, 8, 1}; }
// Step kernel: three CTAs an SM; a unit is a page.
Grid step_grid() { return Grid{kPage, 8, 148 * 3, 4, 2, 32, 16, 1}; }
// Tile kernel: one CTA an SM.  Starting and ending an item takes 7 to 8 us,
// a tile of 128 keys 1 us for up to 128 rows and 2 us for 256.
Grid tile_grid(bool wide, bool int8) {
    if (wide && !int8) return Grid{64, 128, 148, 6, 3, 4, 128, 1};
    return Grid{128, wide ? 128 : 256, 148, 8, 3, 2, 128, 2};
}

Block block_of(const qb_paged_step &s, const Grid &g, int seq, int kvh, int row0, int rows, int G) {
    Block b{seq, kvh, row0, rows, 0, 0, 0, 0, 0};
    const int64_t start = s.starts[seq], lo = start + row0 / G, hi = start + (row0 + rows - 1) / G + 1;
    int64_t w0 = 0, sk = 0;
    if (s.window && lo + 1 > (int64_t)s.window) {
        w0 = lo + 1 - (int64_t)s.window;
        sk = std::min<int64_t>((int64_t)std::min<size_t>(s.sinks, (size_t)INT32_MAX), w0);
    }
    const int64_t end = (hi + g.unit - 1) / g.unit, first = w0 / g.unit, sunits = (sk + g.unit - 1) / g.unit;
    if (sk && sunits < first) {
        b.ns = (int32_t)sunits;
        b.u0 = (int32_t)first;
        b.units = (int32_t)(sunits + end - first);
    } else {
        b.u0 = sk ? 0 : (int32_t)first;
        b.units = (int32_t)(end - b.u0);
    }
    b.w0 = (int32_t)w0;
    b.hi = (int32_t)hi;
    return b;
}

// A way to cut a list of blocks.
enum Cut {
    kWhole,   // not at all
    kEven,    // each block into equal pieces of at most T units
    kStream,  // all blocks in one row, cut every T units
    kTail     // the last `tail` blocks (the shortest) into pieces of at most T units
};

// The lengths of a block's pieces, appended to `out`.  `pos`: units in front
// of the block (kStream); `tail`: one of the last blocks (kTail).
void pieces_of(int units, const Grid &g, Cut how, int T, int64_t pos, bool tail, std::vector<int> &out) {
    int n = 1;
    if (how == kEven || (how == kTail && tail)) n = (units + T - 1) / T;
    if (how != kStream) {
        for (int i = 0; i < n; ++i) out.push_back(units / n + (i < units % n));
        return;
    }
    while (units > 0) {
        int u = (int)(T - pos % T);
        // No piece shorter than `least`: the first takes the next's share
        // too, and a short rest goes with the last.
        if (u < g.least) u += T;
        if (u + g.least > units) u = units;
        out.push_back(u);
        units -= u;
        pos += u;
    }
}

inline int cost_of(const Block &b, const Grid &g, int units, bool part) {
    const int w = b.rows > g.narrow ? g.wide : 1;
    return units * w + g.fixed + (part ? g.part * w : 0);
}

// When every piece is done, with the longest started first on the first free
// slot (what the hardware does with a grid in this order).
double makespan(const std::vector<Block> &bl, const Grid &g, Cut how, int T, size_t tail) {
    std::vector<int> cost, n;
    int64_t total = 0, pos = 0;
    for (size_t i = 0; i < bl.size(); ++i) {
        n.clear();
        pieces_of(bl[i].units, g, how, T, pos, i + tail >= bl.size(), n);
        pos += bl[i].units;
        for (int u : n) {
            cost.push_back(cost_of(bl[i], g, u, n.size() > 1));
            total += cost.back();
        }
    }
    std::sort(cost.begin(), cost.end(), std::greater<int>());
    if (cost.size() <= (size_t)g.slots) return cost[0];
    // Too many to follow one by one: the last wave is ragged by about a
    // short piece.
    if (cost.size() > 4096) return (double)total / g.slots + cost[cost.size() * 7 / 8];
    std::priority_queue<int64_t, std::vector<int64_t>, std::greater<int64_t>> free_at;
    int64_t last = 0;
    for (size_t i = 0; i < cost.size(); ++i) {
        int64_t at = 0;
        if (i >= (size_t)g.slots) {
            at = free_at.top();
            free_at.pop();
        }
        free_at.push(at + cost[i]);
        last = std::max(last, at + cost[i]);
    }
    return (double)last;
}

// Cuts the blocks' units into items (longest first) and lists the merges:
// of a few candidate cuts the one whose simulated end comes first, whole
// blocks if none is clearly better.
void cut(std::vector<Block> &bl, const Grid &g, int hd, bool quads, int64_t &ws, std::vector<Item> &items,
         std::vector<Merge> &merges) {
    if (bl.empty()) return;
    std::stable_sort(bl.begin(), bl.end(), [&](const Block &a, const Block &b) {
        return cost_of(a, g, a.units, false) > cost_of(b, g, b.units, false);
    });
    int64_t total = 0;
    for (const Block &b : bl) total += b.units;
    Cut how = kWhole;
    int T = 1;
    size_t tail = 0;
    double end = makespan(bl, g, kWhole, 1, 0);
    // Whole blocks that fill the slots many times over end evenly anyway.
    if (bl.size() < 8 * (size_t)g.slots || (double)bl[0].units > 0.25 * end) {
        auto consider = [&](Cut h, int t, size_t m) {
            const double e = makespan(bl, g, h, t, m);
            if (e < 0.98 * end) {
                end = e;
                how = h;
                T = t;
                tail = m;
            }
        };
        int before = 0;
        for (double k : {0.7, 0.85, 1.0, 1.25, 1.5, 2.0, 3.0, 4.0, 6.0}) {
            const int t = std::max<int>(g.least, (int)ceil((double)total / (g.slots * k)));
            if (t == before || t >= bl[0].units) continue;
            before = t;
            consider(kEven, t, 0);
            if (k <= 2.0) consider(kStream, t, 0);
        }
        // The blocks of the last, partly filled wave.
        if (const size_t m = bl.size() % g.slots; m && bl.size() > (size_t)g.slots)
            for (int t : {4, 8, 16}) consider(kTail, std::max(g.least, bl.back().units / t), m);
    }
    std::vector<int> n;
    int64_t pos = 0;
    for (size_t i = 0; i < bl.size(); ++i) {
        const Block &b = bl[i];
        n.clear();
        pieces_of(b.units, g, how, T, pos, i + tail >= bl.size(), n);
        pos += b.units;
        const bool part = n.size() > 1;
        const int stride = (b.rows * (hd + 2) + 3) / 4 * 4;
        if (part) merges.push_back(Merge{b.seq, b.kvh, b.row0, b.rows, (int32_t)ws, (int32_t)n.size(), stride, quads});
        int at = 0;
        for (int u : n) {
            items.push_back(Item{b.seq, b.kvh, b.row0, b.rows, at, at + u, b.ns, b.u0, b.w0, b.hi,
                                 part ? (int32_t)ws : -1, cost_of(b, g, u, part)});
            if (part) ws += stride;
            at += u;
        }
    }
    std::stable_sort(items.begin(), items.end(), [](const Item &a, const Item &b) { return a.cost > b.cost; });
}

uint32_t invalid(size_t buffer, size_t expected, size_t actual, size_t index, uint32_t status) {
    set_detail(buffer, expected, actual, index);
    return status;
}

uint32_t build(const qb_paged_step &s, int32_t *words, size_t capacity, qb_paged_plan *out) {
    if (!s.sequences || !s.pages_per_sequence || !s.pages || !s.kv_heads || !s.head_dim || !s.query_heads)
        return QB_ZERO_DIMENSION;
    if (s.value_dtype > QB_PAGED_BF16 || s.cache_dtype > QB_PAGED_INT8) return QB_UNSUPPORTED;
    if (s.query_heads % s.kv_heads || s.head_dim > (size_t)kMaxHeadDim) return QB_INVALID_SHAPE;
    size_t n, rows = 0;
    if (mul_ovf(s.pages, s.kv_heads, &n) || mul_ovf(n, (size_t)kPage, &n) || n > 0x7fffffffu ||
        mul_ovf(s.sequences, s.pages_per_sequence, &n) || n > 0x0fffffffu || s.query_heads > 0xffffu ||
        s.window > 0x7fffffffu)
        return QB_DIMENSION_OVERFLOW;
    if (!s.tables || !s.starts || !s.counts || !out || (capacity && !words)) return QB_INVALID_PARAMETERS;
    size_t tokens = 0;
    for (size_t i = 0; i < s.sequences; ++i) {
        const size_t end = (size_t)s.starts[i] + s.counts[i];
        if (s.counts[i] && end > s.pages_per_sequence * kPage)
            return invalid(1, s.pages_per_sequence * kPage, end, i, QB_FULL);
        tokens += s.counts[i];
    }
    if (!tokens) return QB_ZERO_DIMENSION;
    if (mul_ovf(tokens, s.query_heads, &rows) || rows > 0x3fffffffu ||
        s.pages_per_sequence > 0x07fffff0u)  // (a tile past the last position is still an int32)
        return QB_DIMENSION_OVERFLOW;
    // Every page that a call of this plan touches: what the new tokens see
    // and what they are.  Entries of pages that left the window are not read.
    std::vector<int32_t> written;
    for (size_t i = 0; i < s.sequences; ++i) {
        if (!s.counts[i]) continue;
        const int32_t *t = s.tables + i * s.pages_per_sequence;
        const size_t start = s.starts[i], end = start + s.counts[i];
        const size_t w0 = s.window && start + 1 > s.window ? start + 1 - s.window : 0;
        const size_t sk = std::min(s.sinks, w0);
        for (size_t j = 0; j < (end + kPage - 1) / kPage; ++j) {
            if ((j + 1) * kPage <= w0 && j * kPage >= sk) continue;
            if (t[j] < 0 || (size_t)t[j] >= s.pages)
                return invalid(0, s.pages, (size_t)(uint32_t)t[j], i * s.pages_per_sequence + j, QB_INVALID_PARAMETERS);
        }
        for (size_t j = start / kPage; j < (end + kPage - 1) / kPage; ++j) written.push_back(t[j]);
    }
    std::sort(written.begin(), written.end());
    const bool twice = std::adjacent_find(written.begin(), written.end()) != written.end();

    const int G = (int)(s.query_heads / s.kv_heads), hd = (int)s.head_dim;
    const bool wide = s.value_dtype == QB_PAGED_F32;
    const bool fast = (hd == 64 || hd == 128) && s.cache_dtype != QB_PAGED_F32;
    const Grid small = fast ? step_grid() : rows_grid();
    const Grid tile = tile_grid(wide, s.cache_dtype == QB_PAGED_INT8);
    // Two n8 tiles a block only where some sequence of the list has use for them.
    int nt = 1;
    if (fast)
        for (size_t i = 0; i < s.sequences; ++i)
            if (s.counts[i] * (size_t)G > 8 && s.counts[i] * (size_t)G <= (size_t)kStepRows) nt = 2;
    std::vector<Block> bs, bt;
    for (size_t i = 0; i < s.sequences; ++i) {
        const int64_t r = (int64_t)s.counts[i] * G;
        const bool to_tile = fast && r > kStepRows;
        const Grid &g = to_tile ? tile : small;
        const int64_t step = to_tile ? g.block : fast ? 8 * nt : g.block;
        for (size_t h = 0; h < s.kv_heads; ++h)
            for (int64_t r0 = 0; r0 < r; r0 += step)
                (to_tile ? bt : bs).push_back(block_of(s, g, (int)i, (int)h, (int)r0, (int)std::min(step, r - r0), G));
    }
    std::vector<Item> si, ti;
    std::vector<Merge> merges;
    int64_t ws = 0;
    cut(bs, small, hd, false, ws, si, merges);
    cut(bt, tile, hd, true, ws, ti, merges);
    if (ws > 0x7fffffff) return QB_RESOURCE_BUDGET;

    qb_paged_plan p = {};
    p.sequences = s.sequences;
    p.pages_per_sequence = s.pages_per_sequence;
    p.tokens = tokens;
    p.pages = s.pages;
    p.query_heads = s.query_heads;
    p.kv_heads = s.kv_heads;
    p.head_dim = s.head_dim;
    p.window = s.window;
    p.sinks = s.sinks;
    p.value_dtype = s.value_dtype;
    p.cache_dtype = s.cache_dtype;
    p.workspace_bytes = (size_t)ws * 4;
    p.shared_rows = twice;
    p.small_kind = fast ? (uint32_t)nt : 0u;
    p.small_unit = (uint32_t)small.unit;
    p.tile_unit = (uint32_t)tile.unit;
    p.small_items = (uint32_t)si.size();
    p.tile_items = (uint32_t)ti.size();
    p.merges = (uint32_t)merges.size();
    for (const Merge &m : merges)
        p.merge_blocks = std::max(p.merge_blocks, (uint32_t)(m.parts > kMergeFew ? m.rows : (m.rows + kMergeWarps - 1) / kMergeWarps));
    // Records of 4 words and more start on 16 bytes.
    size_t at = 0;
    auto take = [&](size_t words_) {
        const size_t a = at;
        at += (words_ + 3) / 4 * 4;
        return a;
    };
    const size_t o_seq = take(4 * s.sequences), o_table = take(s.sequences * s.pages_per_sequence),
                 o_slot = take(tokens), o_small = take(12 * si.size()), o_tile = take(12 * ti.size()),
                 o_merge = take(8 * merges.size());
    if (at > 0x7fffffffu) return QB_DIMENSION_OVERFLOW;
    p.words = at;
    p.off_seqs = (uint32_t)o_seq;
    p.off_slots = (uint32_t)o_slot;
    p.off_small = (uint32_t)o_small;
    p.off_tile = (uint32_t)o_tile;
    p.off_merges = (uint32_t)o_merge;
    if (capacity < at) return invalid(2, at, capacity, 0, QB_INVALID_LENGTH);
    size_t tok = 0;
    for (size_t i = 0; i < s.sequences; ++i) {
        const SeqRec r{(int32_t)tok, (int32_t)s.counts[i], (int32_t)s.starts[i],
                       (int32_t)(o_table + i * s.pages_per_sequence)};
        memcpy(words + o_seq + 4 * i, &r, sizeof r);
        const int32_t *t = s.tables + i * s.pages_per_sequence;
        for (size_t j = 0; j < s.counts[i]; ++j, ++tok) {
            const size_t pos = s.starts[i] + j;
            words[o_slot + tok] = t[pos / kPage] * kPage + (int32_t)(pos % kPage);
        }
    }
    memcpy(words + o_table, s.tables, s.sequences * s.pages_per_sequence * sizeof(int32_t));
    if (!si.empty()) memcpy(words + o_small, si.data(), si.size() * sizeof(Item));
    if (!ti.empty()) memcpy(words + o_tile, ti.data(), ti.size() * sizeof(Item));
    if (!merges.empty()) memcpy(words + o_merge, merges.data(), merges.size() * sizeof(Merge));
    *out = p;
    return QB_OK;
}

}  // namespace
}  // namespace paged
}  // namespace qb

using namespace qb;

extern "C" {

uint32_t qb_paged_plan_build(const qb_paged_step *step, int32_t *words, size_t capacity, qb_paged_plan *out) {
    clear_detail();
    if (!step) return QB_INVALID_PARAMETERS;
    try {
        return paged::build(*step, words, capacity, out);
    } catch (const std::bad_alloc &) {
        return QB_ALLOCATION;
    } catch (...) {
        return QB_INVALID_PARAMETERS;
    }
}

}  // extern "C"
