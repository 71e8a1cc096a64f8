// Attention over the paged cache: hfk_prompt_attention and hfk_prefix_attention of include/hfk.h.
//
// Both kernels compute the transposed products  S^T = K Q^T  and  O^T = V^T P^T. A lane then holds scores of one query row
// (the column lane % 32, or lane % 16) and the accumulator's row order is the order in which the second product
// may take its keys, so the weights go from the first product's result registers into the second one's operand without
// crossing lanes; only V has to be transposed. The softmax runs in one pass with a running maximum and sum per
// row, in 32 bits and base 2.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "hfk.h"
#include "hfk_attention_plan.h"
#include "hfk_cache_types.h"

namespace {

using hfk::BlockSplit;
using hfk::f32x16;
using hfk::f32x4;
using hfk::u32x2;
using hfk::u32x4;

constexpr float kMinusInf = -__builtin_huge_valf();
constexpr float kLn2 = 0.693147180559945309f;
constexpr uint32_t kWideThreads = hfk::kWideRows * 2;     // a wave has 32 rows

// One side of the cache for one call; strides in bytes (scales: in floats).
struct CacheSide {
    const char* values;
    const float* scales;
    int64_t block, token, head;
    int64_t scale_block, scale_token, scale_head;
};

struct AttentionArgs {
    CacheSide k, v;
    uint32_t blocks;
    BlockSplit split;
    const char* q;
    char* out;
    float* lse;
    int64_t q_token, q_head, out_token, out_head;   // bytes
    uint32_t n_rows;          // tokens
    uint32_t cache_heads, group, dim;
    float score_scale;        // scale * log2 e
    float* part_sum;          // NULL: the one split writes the result itself
    float* part_stat;         // largest score, sum of weights
};

// What one launch walks: sequences of query rows with their keys.
struct Walk {
    const int64_t* table;     // [n_seqs][width]
    uint32_t width;
    const int64_t* starts;    // [n_seqs + 1], or NULL: sequence b owns `tokens_per_seq` tokens from b * tokens_per_seq
    const int64_t* lens;
    uint32_t n_seqs, tokens_per_seq;
    uint32_t causal;
    uint32_t tiles;           // of query rows: all sequences' (wide), or per sequence (narrow)
    uint32_t splits, chunk;   // chunk: keys per split (narrow)
    uint32_t first_split;     // place of split 0 in the workspace
    uint32_t groups;          // workgroups
};

__device__ uint32_t clamp_len(int64_t len, uint32_t width, uint32_t T) {
    const int64_t most = (int64_t)width * T;
    return (uint32_t)(len < 0 ? 0 : len > most ? most : len);
}

// Both values of a pair of lanes 32 (16) apart, in both of them.
__device__ float max_across_32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ float sum_across_32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ float max_across_16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ float sum_across_16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T, typename V>
__device__ typename T::Vec8 as_vec8(V v) {
    return __builtin_bit_cast(typename T::Vec8, v);
}

__device__ int64_t place(const CacheSide& s, uint32_t block, uint32_t at) { return (int64_t)block * s.block + (int64_t)at * s.token; }
__device__ int64_t scale_place(const CacheSide& s, uint32_t block, uint32_t at) {
    return (int64_t)block * s.scale_block + (int64_t)at * s.scale_token;
}

// ---- wide -------------------------------------------------------------------------------------

// Which rows a workgroup has: tile `tile` of all the sequences' tiles of ROWS rows.
struct Tile {
    uint32_t seq, first_token, tokens, first_row;
    bool found;
};

template <uint32_t ROWS>
__device__ Tile find_tile(const AttentionArgs& a, const Walk& w, uint32_t tile) {
    Tile t{0, 0, 0, 0, false};
    if (w.starts == nullptr) {
        t.tokens = w.tokens_per_seq;
        t.first_row = tile * ROWS;
        t.found = t.first_row < t.tokens * a.group;
        return t;
    }
    const uint32_t lane = threadIdx.x % 64u;
    uint32_t before = 0;
    for (uint32_t base = 0; base < w.n_seqs; base += 64u) {       // 64 sequences at a time, by every wave alike
        const uint32_t b = base + lane;
        int64_t first = 0, last = 0;
        if (b < w.n_seqs) {
            first = w.starts[b];
            last = w.starts[b + 1];
        }
        const bool sound = first >= 0 && last > first && last <= (int64_t)a.n_rows;
        const uint32_t tokens = sound ? (uint32_t)(last - first) : 0u;
        const uint32_t mine = (tokens * a.group + ROWS - 1u) / ROWS;
        uint32_t upto = mine;
        for (uint32_t o = 1; o < 64u; o <<= 1) {
            const uint32_t other = __shfl_up(upto, o);
            if (lane >= o) upto += other;
        }
        const uint64_t past = __ballot(before + upto > tile);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            t.seq = base + at;
            t.first_token = __builtin_amdgcn_readlane((uint32_t)first, at);
            t.tokens = __builtin_amdgcn_readlane(tokens, at);
            t.first_row = (tile - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at))) * ROWS;
            t.found = true;
            return t;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return t;
}

// Rows of K and V in LDS, bytes. Their paddings let a wave read 16 bytes of 16 consecutive keys (K), and 64 bytes of four
// (V, through the transposing read), without two lanes meeting at a bank; every read of a lane then lies at a constant
// distance from one address.
template <int DP>
constexpr uint32_t kKeyRow = DP * 2 + 16;
template <int DP>
constexpr uint32_t kValueRow = DP * 2 + 64;

template <int KEYS>
struct TileKeys {             // where the keys of one tile lie; one that is not visible gets the cache's first token's place
    int64_t k[KEYS], v[KEYS];
    uint64_t seen;            // bit per visible key
};
template <int KEYS>
struct TileScales {
    int64_t k[KEYS], v[KEYS];
};

// Four 16-bit rows' columns: lane i of 16 gets column i of the 4 x 16 values that the 16 lanes point at.
__device__ u32x2 read_transposed(uint32_t lds_byte) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* Lds;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)lds_byte));
}
__device__ u32x4 read_lds(uint32_t lds_byte) {
    typedef __attribute__((address_space(3))) const u32x4* Lds;
    return *(Lds)lds_byte;
}
__device__ uint32_t lds_address(const void* p) {
    typedef __attribute__((address_space(3))) const void* Lds;
    return (uint32_t)(uintptr_t)(Lds)p;
}
// Keeps an address as one register: what is added to it later stays a constant in the instruction, instead of one hoisted
// register for every read of an unrolled loop.
__device__ uint32_t one_register(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

template <typename T, bool FP8, int DP, int KEYS>
__global__ __launch_bounds__(kWideThreads, 2) void wide_attention_kernel(const AttentionArgs a, const Walk w) {
    constexpr uint32_t kRows = hfk::kWideRows, kThreads = kWideThreads, kWaves = kThreads / 64;
    constexpr uint32_t kPieces = FP8 ? DP / 16 : DP / 8;                  // 16-byte pieces of a cached row
    constexpr uint32_t kLoads = (KEYS * kPieces + kThreads - 1) / kThreads;
    constexpr uint32_t kKeyStage = KEYS * kKeyRow<DP>, kValueStage = KEYS * kValueRow<DP>;
    constexpr uint32_t kRing = 8;                                         // tiles whose places are kept
    __shared__ __align__(16) char k_lds[3 * kKeyStage];
    __shared__ __align__(16) char v_lds[3 * kValueStage];
    __shared__ TileKeys<KEYS> keys[kRing];
    __shared__ TileScales<FP8 ? KEYS : 1> scales[kRing];
    __shared__ uint32_t not_finite;

    const uint32_t tid = threadIdx.x, lane = tid % 64u, wave = __builtin_amdgcn_readfirstlane(tid / 64u), col = lane % 32u, half = lane / 32u;
    const uint32_t head = blockIdx.x % a.cache_heads, rest = blockIdx.x / a.cache_heads;
    const uint32_t split = rest % w.splits;
    const Tile t = find_tile<kRows>(a, w, w.tiles - 1u - rest / w.splits);   // long tiles of a causal walk first
    if (!t.found) return;

    const uint32_t n_tile_rows = t.tokens * a.group;
    const uint32_t len = clamp_len(w.lens[t.seq], w.width, a.split.T);
    // Keys that a token sees: all, or (causal) so many that the last token sees all.
    const auto seen_by = [&](uint32_t token) -> int32_t {
        if (!w.causal) return (int32_t)len;
        const int32_t n = (int32_t)len - (int32_t)(t.tokens - 1u - token);
        return n < 0 ? 0 : n;
    };
    const uint32_t last_row = (t.first_row + kRows < n_tile_rows ? t.first_row + kRows : n_tile_rows) - 1u;
    const uint32_t most = (uint32_t)seen_by(last_row / a.group);
    uint32_t first_key = 0, end_key = most;
    if (w.splits > 1) {
        uint32_t span = (most + w.splits - 1u) / w.splits;
        span = (span < hfk::kMinSplitKeys ? hfk::kMinSplitKeys : span) + KEYS - 1u;
        span -= span % KEYS;
        const uint64_t from = (uint64_t)split * span;
        first_key = from < most ? (uint32_t)from : most;
        end_key = most - first_key < span ? most : first_key + span;
    }

    // This lane's query row, and whether its wave has any.
    const uint32_t wave_row = t.first_row + wave * 32u, row = wave_row + col;
    const bool any_row = wave_row < n_tile_rows, owns = row < n_tile_rows;
    const uint32_t local = owns ? row / a.group : 0u, token = t.first_token + local, q_head = head * a.group + (owns ? row % a.group : 0u);
    const int32_t limit = owns ? seen_by(local) : 0;
    typename T::Vec8 q[DP / 16];
    {
        const char* src = a.q + (int64_t)token * a.q_token + (int64_t)q_head * a.q_head;
        for (int s = 0; s < DP / 16; ++s) {
            const uint32_t d = s * 16u + half * 8u;
            u32x4 x{0, 0, 0, 0};
            if (owns && d < a.dim) x = *reinterpret_cast<const u32x4*>(src + 2u * d);
            q[s] = as_vec8<T>(x);
        }
    }
    // The fewest keys that a row of the wave, and of the tile, sees.
    const uint32_t wave_least = any_row ? (uint32_t)seen_by(wave_row / a.group) : 0u;
    const uint32_t tile_least = (uint32_t)seen_by(t.first_row / a.group);

    f32x16 o[DP / 32];
    float top = kMinusInf, sum = 0.0f;
    for (int b = 0; b < DP / 32; ++b)
        for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;

    const int64_t* table = w.table + (uint64_t)t.seq * w.width;
    const char* k_base = a.k.values + (int64_t)head * a.k.head;
    const char* v_base = a.v.values + (int64_t)head * a.v.head;
    const float* k_scale_base = FP8 ? a.k.scales + (int64_t)head * a.k.scale_head : nullptr;
    const float* v_scale_base = FP8 ? a.v.scales + (int64_t)head * a.v.scale_head : nullptr;
    const uint32_t n_tiles = (end_key - first_key + KEYS - 1u) / KEYS;

    // Lane l of wave 0 looks up key l of a tile: the table entry is loaded early, the place written late.
    const auto load_entry = [&](uint32_t tile) -> int64_t {
        const uint32_t key = first_key + tile * KEYS + lane;
        return lane < KEYS && key < end_key ? table[a.split.block32(key)] : -1;
    };
    const auto put_keys = [&](uint32_t tile, int64_t entry) {
        const uint32_t key = first_key + tile * KEYS + lane;
        const bool ok = (uint64_t)entry < a.blocks;
        const uint32_t at = key - a.split.block32(key) * a.split.T;
        TileKeys<KEYS>& out = keys[tile % kRing];
        if (lane < KEYS) {
            out.k[lane] = ok ? place(a.k, (uint32_t)entry, at) : 0;
            out.v[lane] = ok ? place(a.v, (uint32_t)entry, at) : 0;
            if constexpr (FP8) {
                scales[tile % kRing].k[lane] = ok ? scale_place(a.k, (uint32_t)entry, at) : 0;
                scales[tile % kRing].v[lane] = ok ? scale_place(a.v, (uint32_t)entry, at) : 0;
            }
        }
        const uint64_t seen = __ballot(ok);
        if (lane == 0) out.seen = seen;
    };

    // Which keys of a tile are visible, as a scalar.
    constexpr uint64_t kAll = KEYS == 64 ? ~0ull : (1ull << (KEYS % 64)) - 1ull;
    const auto as_scalar = [](uint64_t x) -> uint64_t {
        return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32 | __builtin_amdgcn_readfirstlane((uint32_t)x);
    };
    // A tile's keys, or its values, into registers and from there into their stage. A thread has the same piece of every
    // row it moves; pieces beyond head_dim stay zero.
    struct Pieces {
        u32x4 v[kLoads];
        float scale[kLoads];
    };
    static_assert(kThreads % kPieces == 0);
    const uint32_t piece = tid % kPieces, my_key = tid / kPieces;
    const bool moves = piece * (FP8 ? 16u : 8u) < a.dim;
    const auto key_of = [&](uint32_t n) { return n * (kThreads / kPieces) + my_key; };
    Pieces k_reg, v_reg;
    for (uint32_t n = 0; n < kLoads; ++n) {
        k_reg.v[n] = v_reg.v[n] = u32x4{0, 0, 0, 0};
        k_reg.scale[n] = v_reg.scale[n] = 1.0f;
    }
    // Places are read from LDS a turn before the loads that need them.
    struct Places {
        int64_t at[kLoads], scale[FP8 ? kLoads : 1];
    };
    Places k_place, v_place;
    const auto read_places = [&](Places& p, const int64_t* at, const int64_t* scale) {
        for (uint32_t n = 0; n < kLoads; ++n) {
            const uint32_t key = KEYS * kPieces % kThreads != 0 ? key_of(n) % KEYS : key_of(n);
            p.at[n] = at[key];
            if constexpr (FP8) p.scale[n] = scale[key];
        }
    };
    const auto load_pieces = [&](Pieces& p, const Places& from, const char* base, const float* scale_base) {
        if (!moves) return;
        for (uint32_t n = 0; n < kLoads; ++n) {
            if (KEYS * kPieces % kThreads != 0 && key_of(n) >= KEYS) continue;
            p.v[n] = *reinterpret_cast<const u32x4*>(base + from.at[n] + piece * 16u);
            if constexpr (FP8) p.scale[n] = scale_base[from.scale[n]];
        }
    };
    const auto read_k_places = [&](uint32_t tile) { read_places(k_place, keys[tile % kRing].k, scales[tile % kRing].k); };
    const auto read_v_places = [&](uint32_t tile) { read_places(v_place, keys[tile % kRing].v, scales[tile % kRing].v); };
    const auto load_k = [&](Pieces& to) { load_pieces(to, k_place, k_base, k_scale_base); };
    const auto load_v = [&] { load_pieces(v_reg, v_place, v_base, v_scale_base); };
    const auto store_pieces = [&](const Pieces& p, auto put) {
        for (uint32_t n = 0; n < kLoads; ++n) {
            const uint32_t key = key_of(n);
            if (KEYS * kPieces % kThreads != 0 && key >= KEYS) continue;
            if constexpr (FP8) {
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = p.v[n][2 * h], y = p.v[n][2 * h + 1];
                    put(key, 2 * piece + h,
                        u32x4{T::template from_fp8<false>(x, p.scale[n]), T::template from_fp8<true>(x, p.scale[n]),
                              T::template from_fp8<false>(y, p.scale[n]), T::template from_fp8<true>(y, p.scale[n])});
                }
            } else {
                put(key, piece, p.v[n]);
            }
        }
    };
    const auto store_k = [&](uint32_t tile, const Pieces& from) {
        char* to = k_lds + tile % 3u * kKeyStage;
        store_pieces(from, [&](uint32_t key, uint32_t at, u32x4 x) { *reinterpret_cast<u32x4*>(to + key * kKeyRow<DP> + at * 16u) = x; });
    };
    // V of a key that a row does not see meets a weight of zero there, and must be a number for that. Keys that no row sees
    // become zeros; in tiles that some row sees in part, values that are no numbers are taken out here and given to the rows
    // that do see them at the end.
    const auto store_v = [&](uint32_t tile, uint64_t seen) {
        char* to = v_lds + tile % 3u * kValueStage;
        if (seen == kAll && first_key + (tile + 1u) * KEYS <= tile_least) {
            store_pieces(v_reg, [&](uint32_t key, uint32_t at, u32x4 x) { *reinterpret_cast<u32x4*>(to + key * kValueRow<DP> + at * 16u) = x; });
            return;
        }
        bool found = false;
        store_pieces(v_reg, [&](uint32_t key, uint32_t at, u32x4 x) {
            const bool visible = ((seen >> key) & 1u) != 0;
            for (int i = 0; i < 4; ++i) {
                if (!visible) x[i] = 0u;
                if ((x[i] & T::kExponent) == T::kExponent) {
                    x[i] &= 0xffff0000u;
                    found = true;
                }
                if (((x[i] >> 16) & T::kExponent) == T::kExponent) {
                    x[i] &= 0xffffu;
                    found = true;
                }
            }
            *reinterpret_cast<u32x4*>(to + key * kValueRow<DP> + at * 16u) = x;
        });
        if (found) not_finite = 1u;
    };

    // Where this lane reads in a stage.
    const uint32_t k_from = lds_address(k_lds) + col * kKeyRow<DP> + half * 16u;
    const uint32_t v_from = lds_address(v_lds) + (4 * half + (lane & 15u) / 4u) * kValueRow<DP> + (lane & 16u) * 2u + (lane & 3u) * 8u;

    struct Scores {
        f32x16 s[KEYS / 32];
    };
    struct Weights {
        typename T::Vec8 p[KEYS / 16];
    };
    Scores x;
    Weights y;
    const auto first_product = [&](uint32_t tile) {
        for (int b = 0; b < KEYS / 32; ++b)
            for (int i = 0; i < 16; ++i) x.s[b][i] = 0.0f;
        const uint32_t from = one_register(k_from + tile % 3u * kKeyStage);
        for (int d = 0; d < DP / 16; ++d)
            for (int b = 0; b < KEYS / 32; ++b)
                x.s[b] = T::mfma32(as_vec8<T>(read_lds(from + (b * 32u * kKeyRow<DP> + d * 32u))), q[d], x.s[b]);
    };
    const auto hide = [&](uint32_t tile, uint64_t seen) {
        const uint32_t key0 = first_key + tile * KEYS;
        if (key0 + KEYS > wave_least) {
            asm volatile("");      // a branch that most tiles take past all of this, no selects
            const int32_t mine = limit - (int32_t)(key0 + 4u * half);
            for (int b = 0; b < KEYS / 32; ++b)
                for (int i = 0; i < 16; ++i) x.s[b][i] = b * 32 + 8 * (i / 4) + i % 4 < mine ? x.s[b][i] : kMinusInf;
        }
        if (seen != kAll) {
            asm volatile("");
            for (int b = 0; b < KEYS / 32; ++b) {
                const uint32_t mine = (uint32_t)(seen >> (32 * b)) >> (4u * half);
                for (int i = 0; i < 16; ++i) x.s[b][i] = (mine & (1u << (8 * (i / 4) + i % 4))) != 0 ? x.s[b][i] : kMinusInf;
            }
        }
    };
    // The running maximum moves when a score passes it by 2^8, so that most tiles spare the accumulator's rescaling.
    constexpr float kLazily = 8.0f, kLift = T::kMostWeight != 0.0f ? T::kMostWeight - kLazily : 0.0f;
    const float lazily = kLazily / a.score_scale;
    const auto raise = [&]() {
        float high = x.s[0][0];
        for (int b = 0; b < KEYS / 32; ++b)
            for (int i = 0; i < 16; ++i) high = fmaxf(high, x.s[b][i]);
        high = max_across_32(high);
        if (__any(high > top + lazily)) {
            const float now = fmaxf(top, high);
            const float keep = now == kMinusInf ? 1.0f : __builtin_amdgcn_exp2f((top - now) * a.score_scale);
            top = now;
            sum *= keep;
            for (int b = 0; b < DP / 32; ++b)
                for (int i = 0; i < 16; ++i) o[b][i] *= keep;
        }
    };
    const auto weigh = [&]() {
        const float base = top == kMinusInf ? 0.0f : top * a.score_scale - kLift;
        float add = 0.0f;
        for (int b = 0; b < KEYS / 32; ++b)
            for (int h = 0; h < 2; ++h) {
                float e[8];
                for (int i = 0; i < 8; ++i) {
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x.s[b][8 * h + i], a.score_scale, -base));
                    add += e[i];
                }
                y.p[2 * b + h] = as_vec8<T>(u32x4{T::pack2(e[0], e[1]), T::pack2(e[2], e[3]), T::pack2(e[4], e[5]), T::pack2(e[6], e[7])});
            }
        sum += add;
    };
    // Key order of the second product: value j of half h of 16 keys is key (j / 4) * 8 + 4 h + j % 4, as the first
    // product's result registers have it.
    // Its first operands are read a turn early.
    constexpr int kAhead = 6, kSteps = KEYS * DP / 512;
    typename T::Vec8 ahead[kAhead];
    const auto value_columns = [&](uint32_t from, int step) -> typename T::Vec8 {
        const uint32_t at = from + (step / (DP / 32) * 16u * kValueRow<DP> + step % (DP / 32) * 64u);
        const u32x2 low = read_transposed(at), high = read_transposed(at + 8u * kValueRow<DP>);
        return as_vec8<T>(u32x4{low[0], low[1], high[0], high[1]});
    };
    const auto read_ahead = [&](uint32_t tile) {
        const uint32_t from = one_register(v_from + tile % 3u * kValueStage);
        for (int step = 0; step < kAhead; ++step) ahead[step] = value_columns(from, step);
    };
    const auto second_product = [&](uint32_t tile) {
        const uint32_t from = one_register(v_from + tile % 3u * kValueStage);
        for (int step = 0; step < kSteps; ++step) {
            const int b = step % (DP / 32);
            o[b] = T::mfma32(step < kAhead ? ahead[step] : value_columns(from, step), y.p[step / (DP / 32)], o[b]);
        }
    };

    // The waves of a compute unit's four SIMDs come in two halves that take turns: while one half feeds the matrix units
    // (second product of tile i - 1, first product of tile i) the other takes weights on the vector units and moves tiles,
    // then a barrier swaps them. The second half starts one barrier late. A tile is put into its stage by both halves'
    // threads one turn before the first half reads it; the stage, one of three, was last read two turns earlier.
    if (tid == 0) not_finite = 0u;
    if (n_tiles != 0) {
        const bool late = wave >= kWaves / 2;
        if (wave == 0) {      // tiles behind the last show nothing
            int64_t first[6];
            for (uint32_t i = 0; i < 6u; ++i) first[i] = load_entry(i);
            for (uint32_t i = 0; i < 6u; ++i) put_keys(i, first[i]);
        }
        int64_t entry = wave == 0 ? load_entry(6u) : -1;
        __syncthreads();      // not_finite is cleared, too
        uint64_t seen = as_scalar(keys[0].seen), next_seen = keys[1].seen;
        {
            Pieces k_second = k_reg;
            read_k_places(0);
            read_v_places(0);
            load_k(k_reg);
            load_v();
            read_k_places(1);
            load_k(k_second);
            store_k(0, k_reg);
            store_v(0, seen);
            store_k(1, k_second);
        }
        read_k_places(2);
        read_v_places(1);
        load_k(k_reg);
        load_v();
        read_k_places(3);
        read_v_places(2);
        __syncthreads();
        if (late) __syncthreads();
        const auto vector_turn = [&](uint32_t tile) {
            const uint64_t coming = as_scalar(next_seen);
            store_k(tile + 2u, k_reg);
            store_v(tile + 1u, coming);
            // (the look-up's result before the loads are issued: a wait for it would be one for them)
            if (wave == 0) put_keys(tile + 6u, entry);
            load_k(k_reg);
            if (any_row) {
                hide(tile, seen);
                raise();
                read_ahead(tile);
            }
            load_v();
            if (wave == 0) entry = load_entry(tile + 7u);
            read_k_places(tile + 4u);
            read_v_places(tile + 3u);
            next_seen = keys[(tile + 2u) % kRing].seen;
            if (any_row) weigh();
            seen = coming;
        };
        if (any_row) first_product(0);
        __syncthreads();
        vector_turn(0);
        __syncthreads();
        for (uint32_t tile = 1; tile < n_tiles; ++tile) {
            if (any_row) {
                second_product(tile - 1u);
                first_product(tile);
            }
            __syncthreads();
            vector_turn(tile);
            __syncthreads();
        }
        if (any_row) second_product(n_tiles - 1u);
        if (!late) __syncthreads();
    }

    const float total = sum_across_32(sum);
    const uint64_t heads = a.cache_heads * a.group;
    if (owns) {
        const uint64_t place = (uint64_t)token * heads + q_head;
        const float high = top == kMinusInf ? kMinusInf : top * a.score_scale - kLift;
        if (a.part_sum != nullptr) {
            const uint64_t at = (uint64_t)(w.first_split + split) * a.n_rows * heads + place;
            if (half == 0) {
                a.part_stat[2 * at] = high;
                a.part_stat[2 * at + 1] = total;
            }
            if (top != kMinusInf) {
                float* dst = a.part_sum + at * a.dim;
                for (int b = 0; b < DP / 32; ++b)
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t d = b * 32 + 8 * i + 4 * half;
                        if (d < a.dim) *reinterpret_cast<f32x4*>(dst + d) = f32x4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]};
                    }
            }
        } else {
            const float inverse = top == kMinusInf ? 0.0f : 1.0f / total;
            char* dst = a.out + (int64_t)token * a.out_token + (int64_t)q_head * a.out_head;
            for (int b = 0; b < DP / 32; ++b)
                for (int i = 0; i < 4; ++i) {
                    const uint32_t d = b * 32 + 8 * i + 4 * half;
                    if (d < a.dim)
                        *reinterpret_cast<u32x2*>(dst + 2u * d) = u32x2{T::pack2(o[b][4 * i] * inverse, o[b][4 * i + 1] * inverse),
                                                                      T::pack2(o[b][4 * i + 2] * inverse, o[b][4 * i + 3] * inverse)};
                }
            if (a.lse != nullptr && half == 0) a.lse[place] = top == kMinusInf ? kMinusInf : (high + __log2f(total)) * kLn2;
        }
    }

    // Rare and slow: what was taken out of V, to every row that sees the key it belongs to.
    __syncthreads();
    if (n_tiles == 0 || not_finite == 0) return;
    const uint32_t whole = tile_least > first_key ? (tile_least - first_key) / KEYS * KEYS : 0u;    // keys of untouched tiles
    for (uint32_t n = tid; n < kRows * a.dim; n += kThreads) {
        const uint32_t r = t.first_row + n / a.dim, d = n % a.dim;
        if (r >= n_tile_rows) break;
        const uint32_t of = r / a.group, of_head = head * a.group + r % a.group;
        const uint32_t until = (uint32_t)seen_by(of) < end_key ? (uint32_t)seen_by(of) : end_key;
        float add = 0.0f;
        for (uint32_t key = first_key + whole; key < until; ++key) {
            const uint32_t block = a.split.block32(key), at = key - block * a.split.T;
            const int64_t entry = table[block];
            if ((uint64_t)entry >= a.blocks) continue;
            const char* src = v_base + place(a.v, (uint32_t)entry, at);
            uint32_t bits;
            if constexpr (FP8) bits = T::template from_fp8<false>(reinterpret_cast<const uint8_t*>(src)[d], v_scale_base[scale_place(a.v, (uint32_t)entry, at)]) & 0xffffu;
            else bits = reinterpret_cast<const uint16_t*>(src)[d];
            if ((bits & T::kExponent) == T::kExponent) add += T::to_float(bits);
        }
        if (add == 0.0f) continue;
        const uint64_t at_token = t.first_token + of;
        if (a.part_sum != nullptr) a.part_sum[((uint64_t)(w.first_split + split) * a.n_rows * heads + at_token * heads + of_head) * a.dim + d] = add;
        else reinterpret_cast<uint16_t*>(a.out + (int64_t)at_token * a.out_token + (int64_t)of_head * a.out_head)[d] = (uint16_t)T::pack2(add, add);
    }
}

// ---- narrow -----------------------------------------------------------------------------------

template <typename T, bool FP8, int DP, int R>
__global__ __launch_bounds__(256) void narrow_attention_kernel(const AttentionArgs a, const Walk prefix, const Walk own) {
    constexpr int kKSteps = DP / 32;        // matrix instructions of the first product
    constexpr int kCols = DP / 16;          // values of V per lane and key
    constexpr uint32_t kRegs = R * kCols * 4;
    constexpr float kLift = T::kMostWeight;
    __shared__ float tops[4][R * 16], sums[4][R * 16];
    __shared__ float o_lds[2][kRegs * 64];

    const uint32_t tid = threadIdx.x, lane = tid % 64u, wave = tid / 64u, col = lane % 16u, quarter = lane / 16u;
    const bool is_prefix = blockIdx.x < prefix.groups;
    const Walk& w = is_prefix ? prefix : own;
    const uint32_t group_id = is_prefix ? blockIdx.x : blockIdx.x - prefix.groups;
    const uint32_t head = group_id % a.cache_heads, rest = group_id / a.cache_heads;
    const uint32_t split = rest % w.splits, tile = rest / w.splits % w.tiles, seq = rest / w.splits / w.tiles;

    const uint32_t len = clamp_len(w.lens[seq], w.width, a.split.T);
    const uint64_t from = (uint64_t)split * w.chunk;
    const uint32_t first_key = from < len ? (uint32_t)from : len;
    const uint32_t end_key = len - first_key < w.chunk ? len : first_key + w.chunk;
    const uint32_t n_tile_rows = w.tokens_per_seq * a.group;

    uint32_t token[R], q_head[R];
    bool owns[R];
    typename T::Vec8 q[R][kKSteps];
    for (int r = 0; r < R; ++r) {
        const uint32_t row = (tile * R + r) * 16u + col;
        owns[r] = row < n_tile_rows;
        token[r] = seq * w.tokens_per_seq + (owns[r] ? row / a.group : 0u);
        q_head[r] = head * a.group + (owns[r] ? row % a.group : 0u);
        const char* src = a.q + (int64_t)token[r] * a.q_token + (int64_t)q_head[r] * a.q_head;
        for (int s = 0; s < kKSteps; ++s) {
            // an e4m3 row is loaded 16 values at a time, which two steps share
            const uint32_t d = FP8 ? (s / 2) * 64u + quarter * 16u + (s % 2) * 8u : s * 32u + quarter * 8u;
            u32x4 x{0, 0, 0, 0};
            if (owns[r] && d < a.dim) x = *reinterpret_cast<const u32x4*>(src + 2u * d);
            q[r][s] = as_vec8<T>(x);
        }
    }
    f32x4 o[R][kCols];
    float top[R], sum[R];
    for (int r = 0; r < R; ++r) {
        top[r] = kMinusInf;
        sum[r] = 0.0f;
        for (int c = 0; c < kCols; ++c) o[r][c] = f32x4{0, 0, 0, 0};
    }

    const int64_t* table = w.table + (uint64_t)seq * w.width;
    const char* k_base = a.k.values + (int64_t)head * a.k.head;
    const char* v_base = a.v.values + (int64_t)head * a.v.head;
    const float* k_scale_base = FP8 ? a.k.scales + (int64_t)head * a.k.scale_head : nullptr;
    const float* v_scale_base = FP8 ? a.v.scales + (int64_t)head * a.v.scale_head : nullptr;
    // One block for four keys in a row when blocks hold a multiple of four.
    const bool by_four = a.split.T % 4u == 0;

    const auto look_up = [&](uint32_t key, uint32_t& block, uint32_t& at) -> bool {
        block = at = 0;
        if (key >= end_key) return false;
        const uint32_t n = a.split.block32(key);
        const int64_t entry = table[n];
        if ((uint64_t)entry >= a.blocks) return false;
        block = (uint32_t)entry;
        at = key - n * a.split.T;
        return true;
    };

    for (uint32_t key0 = first_key + wave * 32u; key0 < end_key; key0 += 128u) {
        // The first product's keys: 16 t + col. A lane without its key reads the cache's first row instead and its scores are
        // masked.
        u32x4 k_reg[2][FP8 ? DP / 64 : DP / 32];
        float k_scale[2];
        uint32_t seen = 0;
        for (int t = 0; t < 2; ++t) {
            uint32_t block, at;
            const bool ok = look_up(key0 + t * 16u + col, block, at);
            seen |= ((uint32_t)__ballot(ok) & 0xffffu) << (16 * t);
            const char* src = k_base + place(a.k, block, at);
            for (int n = 0; n < (FP8 ? DP / 64 : DP / 32); ++n) {
                const uint32_t d = FP8 ? n * 64u + quarter * 16u : n * 32u + quarter * 8u;
                k_reg[t][n] = u32x4{0, 0, 0, 0};
                if (d < a.dim) k_reg[t][n] = *reinterpret_cast<const u32x4*>(src + d * (FP8 ? 1u : 2u));
            }
            if constexpr (FP8) k_scale[t] = k_scale_base[scale_place(a.k, block, at)];
        }
        // The second product's: value j of this quarter is key 16 (j / 4) + 4 quarter + j % 4, in the order in which the first
        // product leaves its scores; this lane has columns col * kCols ..+kCols-1 of all eight.
        constexpr int kWords = FP8 ? kCols / 4 : kCols / 2;
        uint32_t v_reg[8][kWords];
        float v_scale[8];
        const uint32_t d0 = col * kCols;
        for (int t = 0; t < 2; ++t) {
            uint32_t block = 0, at = 0;
            bool ok = false;
            const uint32_t base = key0 + t * 16u + quarter * 4u;
            // four keys from one look-up: the last of them inside the sequence says nothing of the first, so each
            // is asked for its own bit of `seen`
            if (by_four) ok = look_up(base, block, at);
            for (int j = 0; j < 4; ++j) {
                if (!by_four) ok = look_up(base + j, block, at);
                const bool mine = ok && ((seen >> (t * 16u + quarter * 4u + j)) & 1u) != 0;
                const uint32_t place_at = by_four ? at + j : at;
                const int64_t where = mine ? place(a.v, block, place_at) : 0;
                for (int x = 0; x < kWords; ++x) v_reg[4 * t + j][x] = 0;
                if (mine && d0 < a.dim) {
                    const char* src = v_base + where + d0 * (FP8 ? 1u : 2u);
                    if constexpr (kWords == 1) {
                        v_reg[4 * t + j][0] = *reinterpret_cast<const uint32_t*>(src);
                    } else if constexpr (kWords == 2) {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(src);
                        v_reg[4 * t + j][0] = x[0];
                        v_reg[4 * t + j][1] = x[1];
                    } else {
                        for (int y = 0; y < kWords / 4; ++y) {
                            const u32x4 x = *reinterpret_cast<const u32x4*>(src + 16 * y);
                            for (int i = 0; i < 4; ++i) v_reg[4 * t + j][4 * y + i] = x[i];
                        }
                    }
                }
                if constexpr (FP8) v_scale[4 * t + j] = mine ? v_scale_base[scale_place(a.v, block, place_at)] : 1.0f;
            }
        }

        f32x4 s[R][2];
        for (int r = 0; r < R; ++r)
            for (int t = 0; t < 2; ++t) s[r][t] = f32x4{0, 0, 0, 0};
        for (int t = 0; t < 2; ++t)
            for (int n = 0; n < kKSteps; ++n) {
                u32x4 x;
                if constexpr (FP8) {
                    const uint32_t w0 = k_reg[t][n / 2][2 * (n % 2)], w1 = k_reg[t][n / 2][2 * (n % 2) + 1];
                    x = u32x4{T::template from_fp8<false>(w0, k_scale[t]), T::template from_fp8<true>(w0, k_scale[t]),
                              T::template from_fp8<false>(w1, k_scale[t]), T::template from_fp8<true>(w1, k_scale[t])};
                } else {
                    x = k_reg[t][n];
                }
                for (int r = 0; r < R; ++r) s[r][t] = T::mfma16(as_vec8<T>(x), q[r][n], s[r][t]);
            }
        if (seen != 0xffffffffu)
            for (int r = 0; r < R; ++r)
                for (int t = 0; t < 2; ++t)
                    for (int i = 0; i < 4; ++i)
                        if (((seen >> (t * 16u + quarter * 4u + i)) & 1u) == 0) s[r][t][i] = kMinusInf;

        typename T::Vec8 p[R];
        for (int r = 0; r < R; ++r) {
            float high = kMinusInf;
            for (int t = 0; t < 2; ++t)
                for (int i = 0; i < 4; ++i) high = fmaxf(high, s[r][t][i]);
            high = max_across_32(max_across_16(high));
            const float now = fmaxf(top[r], high);
            const float keep = now == kMinusInf ? 1.0f : __builtin_amdgcn_exp2f((top[r] - now) * a.score_scale);
            top[r] = now;
            const float base = now == kMinusInf ? 0.0f : now * a.score_scale - kLift;
            float e[8], add = 0.0f;
            for (int t = 0; t < 2; ++t)
                for (int i = 0; i < 4; ++i) {
                    e[4 * t + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][i], a.score_scale, -base));
                    add += e[4 * t + i];
                }
            sum[r] = sum[r] * keep + add;
            for (int c = 0; c < kCols; ++c) o[r][c] *= keep;
            p[r] = as_vec8<T>(u32x4{T::pack2(e[0], e[1]), T::pack2(e[2], e[3]), T::pack2(e[4], e[5]), T::pack2(e[6], e[7])});
        }
        // Columns 2 w and 2 w + 1 of eight keys out of eight dwords.
        for (int x = 0; x < kCols / 2; ++x) {
            uint32_t two[8];
            for (int j = 0; j < 8; ++j) {
                if constexpr (FP8) two[j] = x % 2 ? T::template from_fp8<true>(v_reg[j][x / 2], v_scale[j]) : T::template from_fp8<false>(v_reg[j][x / 2], v_scale[j]);
                else two[j] = v_reg[j][x];
            }
            u32x4 even, odd;
            for (int i = 0; i < 4; ++i) {
                even[i] = __builtin_amdgcn_perm(two[2 * i + 1], two[2 * i], 0x05040100u);
                odd[i] = __builtin_amdgcn_perm(two[2 * i + 1], two[2 * i], 0x07060302u);
            }
            for (int r = 0; r < R; ++r) {
                o[r][2 * x] = T::mfma16(as_vec8<T>(even), p[r], o[r][2 * x]);
                o[r][2 * x + 1] = T::mfma16(as_vec8<T>(odd), p[r], o[r][2 * x + 1]);
            }
        }
    }

    // The four waves' sums into wave 0's.
    for (int r = 0; r < R; ++r) {
        sum[r] = sum_across_32(sum_across_16(sum[r]));
        if (quarter == 0) {
            tops[wave][r * 16 + col] = top[r];
            sums[wave][r * 16 + col] = sum[r];
        }
    }
    __syncthreads();
    for (int r = 0; r < R; ++r) {
        float all = kMinusInf;
        for (int x = 0; x < 4; ++x) all = fmaxf(all, tops[x][r * 16 + col]);
        const float keep = top[r] == kMinusInf ? 0.0f : __builtin_amdgcn_exp2f((top[r] - all) * a.score_scale);
        float total = 0.0f;
        for (int x = 0; x < 4; ++x) {
            const float one = tops[x][r * 16 + col];
            if (one != kMinusInf) total += sums[x][r * 16 + col] * __builtin_amdgcn_exp2f((one - all) * a.score_scale);
        }
        for (int c = 0; c < kCols; ++c) o[r][c] *= keep;
        top[r] = all;
        sum[r] = total;
    }
    for (uint32_t step = 2; step != 0; step >>= 1) {
        if (wave >= step && wave < 2 * step)
            for (int r = 0; r < R; ++r)
                for (int c = 0; c < kCols; ++c)
                    for (int i = 0; i < 4; ++i) o_lds[wave - step][((r * kCols + c) * 4 + i) * 64 + lane] = o[r][c][i];
        __syncthreads();
        if (wave < step)
            for (int r = 0; r < R; ++r)
                for (int c = 0; c < kCols; ++c)
                    for (int i = 0; i < 4; ++i) o[r][c][i] += o_lds[wave][((r * kCols + c) * 4 + i) * 64 + lane];
        __syncthreads();
    }
    if (wave != 0) return;
    for (int r = 0; r < R; ++r) {
        if (!owns[r]) continue;
        const uint64_t row = (uint64_t)token[r] * (a.cache_heads * a.group) + q_head[r];
        const float high = top[r] == kMinusInf ? kMinusInf : top[r] * a.score_scale - kLift;
        if (a.part_sum != nullptr) {
            const uint64_t at = (uint64_t)(w.first_split + split) * a.n_rows * (a.cache_heads * a.group) + row;
            if (quarter == 0) {
                a.part_stat[2 * at] = high;
                a.part_stat[2 * at + 1] = sum[r];
            }
            if (top[r] == kMinusInf) continue;
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = (quarter * 4u + i) * kCols;
                if (d >= a.dim) continue;
                for (int c = 0; c < kCols; c += 4)
                    *reinterpret_cast<f32x4*>(a.part_sum + at * a.dim + d + c) = f32x4{o[r][c][i], o[r][c + 1][i], o[r][c + 2][i], o[r][c + 3][i]};
            }
        } else {
            const float inverse = top[r] == kMinusInf ? 0.0f : 1.0f / sum[r];
            char* dst = a.out + (int64_t)token[r] * a.out_token + (int64_t)q_head[r] * a.out_head;
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = (quarter * 4u + i) * kCols;
                if (d >= a.dim) continue;
                for (int c = 0; c < kCols; c += 4)
                    *reinterpret_cast<u32x2*>(dst + 2u * (d + c)) = u32x2{T::pack2(o[r][c][i] * inverse, o[r][c + 1][i] * inverse),
                                                                        T::pack2(o[r][c + 2][i] * inverse, o[r][c + 3][i] * inverse)};
            }
            if (a.lse != nullptr && quarter == 0) a.lse[row] = top[r] == kMinusInf ? kMinusInf : (high + __log2f(sum[r])) * kLn2;
        }
    }
}

// ---- join -------------------------------------------------------------------------------------

// One wave per query row: the splits' sums, each brought to the common maximum.
template <typename T>
__global__ __launch_bounds__(256) void join_splits_kernel(const AttentionArgs a, uint32_t splits, const int64_t* starts, uint32_t n_seqs) {
    const uint32_t lane = threadIdx.x % 64u, heads = a.cache_heads * a.group;
    const uint64_t rows = (uint64_t)a.n_rows * heads;
    const uint64_t row = (uint64_t)blockIdx.x * 4u + threadIdx.x / 64u;
    if (row >= rows) return;
    const uint32_t token = (uint32_t)(row / heads), head = (uint32_t)(row % heads);
    if (starts != nullptr) {      // rows of no sequence have no splits and stay as they are
        bool inside = false;
        for (uint32_t b = lane; b < n_seqs; b += 64u) {
            const int64_t first = starts[b], last = starts[b + 1];
            inside |= first >= 0 && last <= (int64_t)a.n_rows && (int64_t)token >= first && (int64_t)token < last;
        }
        if (!__any(inside)) return;
    }
    float high = kMinusInf;
    for (uint32_t s = lane; s < splits; s += 64u) high = fmaxf(high, a.part_stat[2 * (s * rows + row)]);
    for (uint32_t o = 32; o != 0; o >>= 1) high = fmaxf(high, __shfl_xor(high, (int)o));
    float total = 0.0f;
    f32x4 acc{0, 0, 0, 0};
    const uint32_t d = lane * 4u;
    for (uint32_t base = 0; base < splits; base += 64u) {
        float weight = 0.0f;
        if (base + lane < splits) {
            const uint64_t at = (uint64_t)(base + lane) * rows + row;
            const float top = a.part_stat[2 * at];
            if (top != kMinusInf) {
                weight = __builtin_amdgcn_exp2f(top - high);
                total += weight * a.part_stat[2 * at + 1];
            }
        }
        const uint32_t n = splits - base < 64u ? splits - base : 64u;
        for (uint32_t s = 0; s < n; ++s) {
            const float x = __shfl(weight, (int)s);
            if (x == 0.0f) continue;      // nothing was written there, or it vanishes
            if (d < a.dim) acc += x * *reinterpret_cast<const f32x4*>(a.part_sum + ((uint64_t)(base + s) * rows + row) * a.dim + d);
        }
    }
    for (uint32_t o = 32; o != 0; o >>= 1) total += __shfl_xor(total, (int)o);
    const float inverse = high == kMinusInf ? 0.0f : 1.0f / total;
    if (d < a.dim) {
        char* dst = a.out + (int64_t)token * a.out_token + (int64_t)head * a.out_head + 2u * d;
        *reinterpret_cast<u32x2*>(dst) = u32x2{T::pack2(acc[0] * inverse, acc[1] * inverse), T::pack2(acc[2] * inverse, acc[3] * inverse)};
    }
    if (a.lse != nullptr && lane == 0) a.lse[row] = high == kMinusInf ? kMinusInf : (high + __log2f(total)) * kLn2;
}

// ---- host -------------------------------------------------------------------------------------

constexpr uint64_t kMostKeys = 1ull << 30;       // of one sequence

int check_attention(const hfk_attention* a) {
    if (a == nullptr) return HFK_ERR_NULL_POINTER;
    int rc = hfk::check_plane(a->k);
    if (rc == HFK_OK) rc = hfk::check_plane(a->v);
    if (rc == HFK_OK) rc = hfk::check_rows(a->q, a->n_rows);
    if (rc == HFK_OK) rc = hfk::check_rows(a->out, a->n_rows);
    if (rc != HFK_OK) return rc;
    const hfk_cache_plane &k = a->k, &v = a->v;
    if (k.type != v.type || a->out.type != a->q.type || (k.type != HFK_FP8_E4M3 && k.type != a->q.type)) return HFK_ERR_BAD_TYPE;
    if (k.blocks != v.blocks || k.block_tokens != v.block_tokens || k.heads != v.heads || k.head_dim != v.head_dim) return HFK_ERR_BAD_SIZE;
    if (k.head_dim % 16u != 0 || k.head_dim > 256u) return HFK_ERR_BAD_SIZE;
    if (a->q_heads == 0 || a->q_heads % k.heads != 0) return HFK_ERR_BAD_SIZE;
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return HFK_ERR_BAD_SIZE;
    if (a->q_heads > 65535u || a->n_rows > 0x7fffffffull || a->n_rows * a->q_heads > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    if (!hfk::plane_aligned(k, 16) || !hfk::plane_aligned(v, 16) || !hfk::rows_aligned(a->q) || !hfk::rows_aligned(a->out))
        return HFK_ERR_BAD_ALIGNMENT;
    if (a->lse != nullptr && !hfk::multiple_of(a->lse, 4)) return HFK_ERR_BAD_ALIGNMENT;
    return HFK_OK;
}

CacheSide side_of(const hfk_cache_plane& p) {
    const int64_t e = hfk::type_bytes(p.type);
    return {static_cast<const char*>(p.values), p.type == HFK_FP8_E4M3 ? p.scales : nullptr, e * p.block_stride, e * p.token_stride,
            e * p.head_stride, p.scale_block_stride, p.scale_token_stride, p.scale_head_stride};
}

// The workspace holds the splits' sums and, behind them, their maxima and sums of weights.
AttentionArgs fill(const hfk_attention* a, void* workspace, uint64_t splits) {
    AttentionArgs x{};
    x.k = side_of(a->k);
    x.v = side_of(a->v);
    x.blocks = (uint32_t)a->k.blocks;
    x.split = BlockSplit::of(a->k.block_tokens);
    x.q = static_cast<const char*>(a->q.data);
    x.out = static_cast<char*>(a->out.data);
    x.lse = a->lse;
    x.q_token = 2 * a->q.token_stride;
    x.q_head = 2 * a->q.head_stride;
    x.out_token = 2 * a->out.token_stride;
    x.out_head = 2 * a->out.head_stride;
    x.n_rows = (uint32_t)a->n_rows;
    x.cache_heads = a->k.heads;
    x.group = a->q_heads / a->k.heads;
    x.dim = a->k.head_dim;
    x.score_scale = a->scale * 1.44269504088896341f;
    if (splits > 1) {
        x.part_sum = static_cast<float*>(workspace);
        x.part_stat = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                               hfk::round_up(a->n_rows * a->q_heads * splits * a->k.head_dim * 4, 256));
    }
    return x;
}

int check_workspace(void* workspace, uint64_t bytes, uint64_t needed) {
    if (needed == 0) return HFK_OK;
    if (workspace == nullptr) return HFK_ERR_NULL_POINTER;
    if (bytes < needed) return HFK_ERR_WORKSPACE_TOO_SMALL;
    return hfk::multiple_of(workspace, 256) ? HFK_OK : HFK_ERR_BAD_ALIGNMENT;
}

template <typename T, bool FP8>
void launch_wide(const AttentionArgs& x, const Walk& w, hipStream_t s) {
    switch (hfk::padded_head_dim(x.dim)) {
        case 64: wide_attention_kernel<T, FP8, 64, 64><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
        case 128: wide_attention_kernel<T, FP8, 128, 64><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
        default: wide_attention_kernel<T, FP8, 256, 32><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
    }
}

template <typename T, bool FP8, int DP>
void launch_narrow_rows(const AttentionArgs& x, const Walk& prefix, const Walk& own, uint32_t row_blocks, hipStream_t s) {
    const uint32_t grid = prefix.groups + own.groups;
    if (row_blocks == 1) narrow_attention_kernel<T, FP8, DP, 1><<<grid, 256, 0, s>>>(x, prefix, own);
    else if (row_blocks == 2) narrow_attention_kernel<T, FP8, DP, 2><<<grid, 256, 0, s>>>(x, prefix, own);
    else if constexpr (DP != 256) narrow_attention_kernel<T, FP8, DP, 4><<<grid, 256, 0, s>>>(x, prefix, own);
}

template <typename T, bool FP8>
void launch_narrow(const AttentionArgs& x, const Walk& prefix, const Walk& own, uint32_t row_blocks, hipStream_t s) {
    switch (hfk::padded_head_dim(x.dim)) {
        case 64: launch_narrow_rows<T, FP8, 64>(x, prefix, own, row_blocks, s); break;
        case 128: launch_narrow_rows<T, FP8, 128>(x, prefix, own, row_blocks, s); break;
        default: launch_narrow_rows<T, FP8, 256>(x, prefix, own, row_blocks, s); break;
    }
}

template <typename T>
void launch_join(const AttentionArgs& x, uint32_t splits, const int64_t* starts, uint32_t n_seqs, hipStream_t s) {
    const uint64_t rows = (uint64_t)x.n_rows * x.cache_heads * x.group;
    join_splits_kernel<T><<<(uint32_t)((rows + 3) / 4), 256, 0, s>>>(x, splits, starts, n_seqs);
}

int finish() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? HFK_OK : (int)e;
}

// f(element type, is the cache e4m3)
template <typename F>
void by_type(const hfk_attention* a, F f) {
    const bool fp8 = a->k.type == HFK_FP8_E4M3;
    if (a->q.type == HFK_BF16) {
        if (fp8) f(hfk::Bf16{}, std::true_type{});
        else f(hfk::Bf16{}, std::false_type{});
    } else {
        if (fp8) f(hfk::Fp16{}, std::true_type{});
        else f(hfk::Fp16{}, std::false_type{});
    }
}

int most_keys(uint64_t width, uint32_t T, uint64_t& keys) {
    if (width > kMostKeys || width * T > kMostKeys) return HFK_ERR_TOO_LARGE;
    keys = width * T;
    return HFK_OK;
}

}  // namespace

extern "C" {

int hfk_prompt_attention_workspace(const hfk_attention* a, uint64_t n_seqs, uint64_t table_width, uint64_t* bytes) {
    if (bytes == nullptr) return HFK_ERR_NULL_POINTER;
    uint64_t keys = 0;
    int rc = check_attention(a);
    if (rc == HFK_OK) rc = most_keys(table_width, a->k.block_tokens, keys);
    if (rc != HFK_OK) return rc;
    *bytes = hfk::plan_prompt(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, n_seqs, keys).workspace;
    return HFK_OK;
}

int hfk_prompt_attention(const hfk_attention* a, const int64_t* block_table, uint64_t n_seqs, uint64_t table_width,
                         const int64_t* query_starts, const int64_t* kv_lens, int causal, void* workspace,
                         uint64_t workspace_bytes, hfk_stream_t stream) {
    uint64_t keys = 0;
    int rc = check_attention(a);
    if (rc == HFK_OK) rc = most_keys(table_width, a->k.block_tokens, keys);
    if (rc != HFK_OK) return rc;
    if (n_seqs > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    if (n_seqs == 0 || a->n_rows == 0) return HFK_OK;
    if (query_starts == nullptr || kv_lens == nullptr || (table_width != 0 && block_table == nullptr)) return HFK_ERR_NULL_POINTER;
    const hfk::PromptPlan p = hfk::plan_prompt(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, n_seqs, keys);
    rc = check_workspace(workspace, workspace_bytes, p.workspace);
    if (rc != HFK_OK) return rc;
    if (p.wide.groups > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    const AttentionArgs x = fill(a, workspace, p.wide.splits);
    Walk w{};
    w.table = block_table;
    w.width = x.blocks != 0 ? (uint32_t)table_width : 0;      // a cache without blocks shows nothing
    w.starts = query_starts;
    w.lens = kv_lens;
    w.n_seqs = (uint32_t)n_seqs;
    w.causal = causal != 0;
    w.tiles = (uint32_t)p.wide.tiles;
    w.splits = p.wide.splits;
    w.groups = (uint32_t)p.wide.groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(a, [&](auto type, auto fp8) {
        using T = decltype(type);
        launch_wide<T, decltype(fp8)::value>(x, w, s);
        if (w.splits > 1) launch_join<T>(x, w.splits, query_starts, w.n_seqs, s);
    });
    return finish();
}

int hfk_prefix_attention_workspace(const hfk_attention* a, uint64_t n_prefix_blocks, uint64_t table_width, uint64_t* bytes) {
    if (bytes == nullptr) return HFK_ERR_NULL_POINTER;
    uint64_t own = 0, prefix = 0;
    int rc = check_attention(a);
    if (rc == HFK_OK) rc = most_keys(table_width, a->k.block_tokens, own);
    if (rc == HFK_OK) rc = most_keys(n_prefix_blocks, a->k.block_tokens, prefix);
    if (rc != HFK_OK) return rc;
    *bytes = hfk::plan_prefix(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, prefix, own).workspace;
    return HFK_OK;
}

int hfk_prefix_attention(const hfk_attention* a, const int64_t* prefix_blocks, uint64_t n_prefix_blocks,
                         const int64_t* prefix_len, const int64_t* block_table, uint64_t table_width,
                         const int64_t* kv_lens, void* workspace, uint64_t workspace_bytes, hfk_stream_t stream) {
    uint64_t own = 0, prefix = 0;
    int rc = check_attention(a);
    if (rc == HFK_OK) rc = most_keys(table_width, a->k.block_tokens, own);
    if (rc == HFK_OK) rc = most_keys(n_prefix_blocks, a->k.block_tokens, prefix);
    if (rc != HFK_OK) return rc;
    if (a->n_rows == 0) return HFK_OK;
    if (kv_lens == nullptr || (table_width != 0 && block_table == nullptr) ||
        (n_prefix_blocks != 0 && (prefix_blocks == nullptr || prefix_len == nullptr)))
        return HFK_ERR_NULL_POINTER;
    const hfk::PrefixPlan p = hfk::plan_prefix(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, prefix, own);
    rc = check_workspace(workspace, workspace_bytes, p.workspace);
    if (rc != HFK_OK) return rc;
    if (p.wide.groups + p.prefix.groups + p.own.groups > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    const AttentionArgs x = fill(a, workspace, p.splits);
    Walk shared{}, alone{}, none{};
    shared.table = prefix_blocks;
    shared.width = x.blocks != 0 ? (uint32_t)n_prefix_blocks : 0;      // a cache without blocks shows nothing
    shared.lens = prefix_len;
    shared.n_seqs = 1;
    shared.tokens_per_seq = (uint32_t)a->n_rows;
    shared.tiles = (uint32_t)(p.wide_prefix ? p.wide.tiles : p.prefix.row_tiles);
    shared.splits = p.wide_prefix ? p.wide.splits : p.prefix.splits;
    shared.chunk = p.prefix.chunk;
    shared.groups = (uint32_t)(p.wide_prefix ? p.wide.groups : p.prefix.groups);
    alone.table = block_table;
    alone.width = x.blocks != 0 ? (uint32_t)table_width : 0;
    alone.lens = kv_lens;
    alone.n_seqs = (uint32_t)a->n_rows;
    alone.tokens_per_seq = 1;
    alone.tiles = (uint32_t)p.own.row_tiles;
    alone.splits = p.own.splits;
    alone.chunk = p.own.chunk;
    alone.first_split = prefix != 0 ? shared.splits : 0;
    alone.groups = (uint32_t)p.own.groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(a, [&](auto type, auto fp8) {
        using T = decltype(type);
        constexpr bool kFp8 = decltype(fp8)::value;
        if (prefix != 0 && p.wide_prefix) launch_wide<T, kFp8>(x, shared, s);
        if (prefix != 0 && !p.wide_prefix && p.prefix.row_blocks == p.own.row_blocks) {
            launch_narrow<T, kFp8>(x, shared, alone, p.own.row_blocks, s);
        } else {
            if (prefix != 0 && !p.wide_prefix) launch_narrow<T, kFp8>(x, shared, none, p.prefix.row_blocks, s);
            launch_narrow<T, kFp8>(x, none, alone, p.own.row_blocks, s);
        }
        if (p.splits > 1) launch_join<T>(x, p.splits, nullptr, 0, s);
    });
    return finish();
}

}  // extern "C"
