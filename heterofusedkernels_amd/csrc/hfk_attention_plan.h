// Launch planning of the attention entry points: plain C++, no device code, so that it can be checked without a GPU.
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
constexpr uint32_t kMinSplitKeys = 256;    // no split shorter than this: its fixed cost would show

inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
inline uint64_t round_up(uint64_t a, uint64_t b) { return ceil_div(a, b) * b; }
inline uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }
inline uint64_t max64(uint64_t a, uint64_t b) { return a < b ? b : a; }

// Head sizes are served by the next of these, zero-filled beyond head_dim.
inline uint32_t padded_head_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Floats of one row of one split in the workspace: the sum, the largest score (times log2 e), the sum of weights.
inline uint64_t partial_bytes(uint64_t rows, uint64_t splits, uint32_t head_dim) {
    return round_up(rows * splits * head_dim * 4, 256) + round_up(rows * splits * 8, 256);
}

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
    p.splits = (uint32_t)max64(1, min64(ceil_div(wanted_groups, whole), most_keys / kMinSplitKeys));
    p.groups = p.tiles * cache_heads * p.splits;
    return p;
}

struct NarrowPlan {
    uint32_t row_blocks;     // 16 query rows each, per wave: 1, 2 or 4
    uint64_t row_tiles;      // per sequence
    uint32_t chunk;          // keys of one workgroup, a multiple of 128
    uint32_t splits;
    uint64_t groups;
};

// rows: tokens * group of one sequence.
inline NarrowPlan plan_narrow(uint64_t rows, uint64_t n_seqs, uint32_t cache_heads, uint32_t head_dim, uint64_t most_keys,
                              uint64_t wanted_groups) {
    NarrowPlan p{};
    const uint32_t most = padded_head_dim(head_dim) == 256 ? 2 : 4;
    p.row_blocks = rows <= 16 ? 1 : (rows <= 32 || most == 2) ? 2 : 4;
    p.row_tiles = ceil_div(rows, 16ull * p.row_blocks);
    const uint64_t items = max64(1, p.row_tiles * n_seqs * cache_heads);
    p.chunk = (uint32_t)round_up(max64(kMinSplitKeys, ceil_div(most_keys * items, wanted_groups)), 128);
    if (p.chunk > (1u << 30)) p.chunk = 1u << 30;
    p.splits = (uint32_t)max64(1, ceil_div(most_keys, p.chunk));
    p.groups = p.row_tiles * n_seqs * cache_heads * p.splits;
    return p;
}

struct PromptPlan {
    WidePlan wide;
    uint64_t workspace;      // 0: one split, results written directly
};

inline PromptPlan plan_prompt(uint64_t n_rows, uint32_t q_heads, uint32_t cache_heads, uint32_t head_dim, uint64_t n_seqs,
                              uint64_t most_keys) {
    PromptPlan p{};
    p.wide = plan_wide(n_rows * (q_heads / cache_heads), n_seqs, cache_heads, most_keys, 512);
    p.workspace = p.wide.splits > 1 ? partial_bytes(n_rows * q_heads, p.wide.splits, head_dim) : 0;
    return p;
}

struct PrefixPlan {
    bool wide_prefix;        // the prefix goes through the wide kernel (more rows than a narrow workgroup takes)
    WidePlan wide;
    NarrowPlan prefix, own;  // prefix.splits == 0: no narrow prefix
    uint32_t splits;         // of prefix and own tokens together
    uint64_t workspace;
};

inline PrefixPlan plan_prefix(uint64_t n_rows, uint32_t q_heads, uint32_t cache_heads, uint32_t head_dim, uint64_t prefix_keys,
                              uint64_t own_keys) {
    PrefixPlan p{};
    const uint32_t group = q_heads / cache_heads;
    uint32_t prefix_splits = 0;
    if (prefix_keys != 0) {
        p.wide_prefix = n_rows * group > (padded_head_dim(head_dim) == 256 ? 32 : 64);
        if (p.wide_prefix) {
            p.wide = plan_wide(n_rows * group, 1, cache_heads, prefix_keys, 512);
            prefix_splits = p.wide.splits;
        } else {
            p.prefix = plan_narrow(n_rows * group, 1, cache_heads, head_dim, prefix_keys, 1024);
            prefix_splits = p.prefix.splits;
        }
    }
    p.own = plan_narrow(group, n_rows, cache_heads, head_dim, own_keys, 8192);
    p.splits = prefix_splits + p.own.splits;
    p.workspace = p.splits > 1 ? partial_bytes(n_rows * q_heads, p.splits, head_dim) : 0;
    return p;
}

}  // namespace hfk
