// Launch planning of the attention entry points: plain C++, no device code, so that it can be checked without a GPU.
//
// The plans are made for at least one row and one sequence.
//
// Two kernels do the work. The wide one gives a workgroup a tile of query rows (a row is a token and a query head
// of one cache head's group) and walks keys and values through LDS, shared by its waves: many rows per key, bound by
// the matrix units. The narrow one gives every wave of a workgroup its own keys straight from memory for up to 64
// rows: few rows per key, bound by HBM. Where a launch would leave compute units idle the keys are split, every split
// leaves its unnormalised sum, its largest score and its sum of weights in the workspace, and one more launch joins them.
#pragma once
#include <cstdint>

namespace hfk {

constexpr uint32_t kWideRows = 256;        // query rows of a wide workgroup
// No split of a wide workgroup's keys is shorter than this: its fixed cost would show. (Microseconds with 128 | 256 | 512, 32 heads over 8 of
// 128: 33 tokens behind 600: 17.6 | 22.4 | 26.6; 250 behind 1000: 30.3 | 29.9 | 37.2; behind 4000: 40.5 all three. 4 heads over 1 of 64, 250
// behind 2000: 19.3 | 21.5 | 27.3.)
constexpr uint32_t kMinSplitKeys = 256;

// Cache heads of a narrow workgroup's four waves, and the keys they take at a time.
inline uint32_t narrow_heads(uint32_t cache_heads) { return cache_heads % 4 == 0 ? 4 : 1; }
inline uint32_t narrow_unit(uint32_t cache_heads) { return 32 * 4 / narrow_heads(cache_heads); }

inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
inline uint64_t round_up(uint64_t a, uint64_t b) { return ceil_div(a, b) * b; }
inline uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }
inline uint64_t max64(uint64_t a, uint64_t b) { return a < b ? b : a; }

// Head sizes are served by the next of these, zero-filled beyond head_dim.
inline uint32_t padded_head_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Rows of splits in the workspace: a sum each, and behind all of them the largest score (times log2 e) and the sum of weights.
inline uint64_t partial_bytes(uint64_t rows, uint32_t head_dim) { return round_up(rows * head_dim * 4, 256) + round_up(rows * 8, 256); }

struct WidePlan {
    uint64_t tiles;      // upper bound over the sequences: each one's last tile may be partly filled
    uint32_t splits;     // of each tile's keys
    uint64_t groups;     // workgroups
};

// rows: tokens * group, of all sequences together.
inline WidePlan plan_wide(uint64_t rows, uint64_t n_seqs, uint32_t cache_heads, uint64_t most_keys, uint64_t wanted_groups) {
    WidePlan p{};
    p.tiles = rows / kWideRows + min64(n_seqs, rows);
    if (n_seqs == 1) p.tiles = ceil_div(rows, kWideRows);
    const uint64_t whole = max64(1, p.tiles * cache_heads);
    p.splits = (uint32_t)max64(1, min64(wanted_groups / whole, most_keys / kMinSplitKeys));
    p.groups = p.tiles * cache_heads * p.splits;
    return p;
}

struct NarrowPlan {
    uint32_t row_blocks;     // 16 query rows each, per wave: 1, 2 or 4
    uint64_t row_tiles;      // per sequence
    uint32_t ranges;         // shares of all sequences' keys together
    uint64_t groups;
};

// rows: tokens * group of one sequence; units: the most units of keys that all sequences can have together. As many workgroups
// as are resident at once, each with an equal share of the keys there are: rounds of more workgroups than that end ragged.
inline NarrowPlan plan_narrow(uint64_t rows, uint32_t cache_heads, uint32_t head_dim, uint64_t units) {
    NarrowPlan p{};
    const uint32_t dim = padded_head_dim(head_dim), most = dim == 256 ? 2 : 4;
    p.row_blocks = rows <= 16 ? 1 : (rows <= 32 || most == 2) ? 2 : 4;
    p.row_tiles = ceil_div(rows, 16ull * p.row_blocks);
    // Two per compute unit where their registers fit without spilling. (24 sequences of 8000 tokens, 4 heads of 256 in bf16: 149 us
    // with one, 180 with two whose registers spill; one sequence of 32000: 44 and 67 us.)
    const uint64_t resident = p.row_blocks * dim <= 256 && dim != 256 ? 512 : 256, same_keys = p.row_tiles * (cache_heads / narrow_heads(cache_heads));
    uint64_t ranges = min64(max64(1, resident / same_keys), max64(1, units));
    if (ranges > 8) ranges -= ranges % 8;      // the same number for each XCD
    p.ranges = (uint32_t)ranges;
    p.groups = ranges * same_keys;
    return p;
}

// Splits that the parts of n_seqs sequences make (see NarrowWalk).
inline uint64_t own_splits(const NarrowPlan& p, uint64_t n_seqs) { return n_seqs == 1 ? p.ranges : p.ranges + n_seqs; }

struct PromptPlan {
    WidePlan wide;
    uint64_t workspace;      // 0: one split, results written directly
};

inline PromptPlan plan_prompt(uint64_t n_rows, uint32_t q_heads, uint32_t cache_heads, uint32_t head_dim, uint64_t n_seqs,
                              uint64_t most_keys) {
    PromptPlan p{};
    p.wide = plan_wide(n_rows * (q_heads / cache_heads), n_seqs, cache_heads, most_keys, 256);
    p.workspace = p.wide.splits > 1 ? partial_bytes(n_rows * q_heads * p.wide.splits, head_dim) : 0;
    return p;
}

struct PrefixPlan {
    bool wide_prefix;        // the prefix goes through the wide kernel (more rows than a narrow workgroup takes)
    WidePlan wide;
    NarrowPlan prefix, own;
    uint64_t workspace;
};

inline PrefixPlan plan_prefix(uint64_t n_rows, uint32_t q_heads, uint32_t cache_heads, uint32_t head_dim, uint64_t prefix_keys,
                              uint64_t own_keys) {
    PrefixPlan p{};
    const uint32_t group = q_heads / cache_heads;
    if (prefix_keys != 0) {
        // Wide from more rows than one narrow workgroup takes, which would read the prefix again for every tile of rows. Microseconds of
        // a call under 16384 tokens of 8 heads in bf16, rows per cache head: narrow | wide
        //   heads of 64:  16: 22.0 | 26.6, 32: 30.1 | 26.8, 64: 38.8 | 27.4,  96: 42.1 | 28.4, 256:  47.7 |  37.3
        //   heads of 128: 16: 33.5 | 33.0, 32: 44.1 | 33.6, 64: 47.0 | 34.9,  96: 53.4 | 36.7, 256:  68.2 |  46.4
        //   heads of 256: 16: 54.6 | 94.0, 32: 70.6 | 94.9, 64: 75.8 | 99.4, 128: 87.5 | 123,  256: 125   | 195 (wide spills registers)
        // The times cross at fewer rows for heads of up to 128, and not at all here for heads of 256.
        p.wide_prefix = n_rows * group > (padded_head_dim(head_dim) == 256 ? 32 : 64);
        if (p.wide_prefix) p.wide = plan_wide(n_rows * group, 1, cache_heads, prefix_keys, 256);
        else p.prefix = plan_narrow(n_rows * group, cache_heads, head_dim, ceil_div(prefix_keys, narrow_unit(cache_heads)));
        p.workspace += partial_bytes(n_rows * q_heads * (p.wide_prefix ? p.wide.splits : p.prefix.ranges), head_dim);
    }
    p.own = plan_narrow(group, cache_heads, head_dim, n_rows * ceil_div(own_keys, narrow_unit(cache_heads)));
    p.workspace += partial_bytes(own_splits(p.own, n_rows) * q_heads, head_dim);
    return p;
}

}  // namespace hfk
