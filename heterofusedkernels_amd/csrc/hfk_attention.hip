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

// One side of the cache for one call; strides in bytes (scales: in floats). A block spans less than 4 GiB (checked on the
// host), so that a token's place takes 32-bit products; only their sum over blocks is longer.
struct CacheSide {
    const char* values;
    const float* scales;
    int64_t head, scale_head;
    uint32_t block, token;
    uint32_t scale_block, scale_token;
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
};

// Where a launch leaves what the join takes: unnormalised sums [splits][rows][dim], and beside them [splits][rows] pairs of the
// largest score (times log2 e) and the sum of weights. A largest score of -infinity: nothing was seen, no sum was written.
struct Partials {
    float* sum;               // NULL: the one split writes the result itself
    float* stat;
};

// What a wide launch walks: sequences of query rows with their keys.
struct WideWalk {
    const int64_t* table;     // [n_seqs][width]
    uint32_t width;
    const int64_t* starts;    // [n_seqs + 1], or NULL: one sequence that owns all rows
    const int64_t* lens;
    uint32_t n_seqs;
    uint32_t causal;
    uint32_t tiles;           // of query rows, all sequences'
    uint32_t splits;
    uint32_t groups;          // workgroups
    Partials to;
};

// What a narrow launch walks: the keys of n_seqs sequences as one row of units, cut into `ranges` equal shares whatever
// sequences they fall into. Every sequence has tokens_per_seq tokens. A share's part of a sequence is a split.
struct NarrowWalk {
    const int64_t* table;     // [n_seqs][width]
    uint32_t width;
    const int64_t* lens;
    uint32_t n_seqs, tokens_per_seq;
    uint32_t tiles;           // of query rows, per sequence
    uint32_t unit;            // keys: 32 for each wave that works at one head
    uint32_t ranges;
    uint32_t groups;          // workgroups
    // n_seqs == 1: split s is range s and has every row. Else range g's part of sequence b is split g + b, which no other
    // part is (from one part to the next at least one of the two grows), and has b's rows alone.
    Partials to;
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

// The running maximum moves when a score passes it by 2^8, so that most tiles spare the accumulator's rescaling.
constexpr float kLazily = 8.0f;
// Weights of the type T are lifted so that none passes 2^kMostWeight.
template <typename T>
constexpr float kLiftOf = T::kMostWeight != 0.0f ? T::kMostWeight - kLazily : 0.0f;

template <typename T, typename V>
__device__ typename T::Vec8 as_vec8(V v) {
    return __builtin_bit_cast(typename T::Vec8, v);
}

// Eight weights as an operand, and what rounding them to 16 bits took away as another: with a second product of those the
// weights are as good as 32 bits. That one has sums of its own, which count where the first one's are numbers: with V
// infinite it would give NaN where the first gives infinity.
template <typename T>
__device__ typename T::Vec8 pack8(const float (&e)[8]) {
    return as_vec8<T>(u32x4{T::pack2(e[0], e[1]), T::pack2(e[2], e[3]), T::pack2(e[4], e[5]), T::pack2(e[6], e[7])});
}
template <typename T>
__device__ typename T::Vec8 rest8(const float (&e)[8], typename T::Vec8 p) {
    float rest[8];
    for (int i = 0; i < 8; ++i) rest[i] = e[i] - (float)p[i];
    return pack8<T>(rest);
}
__device__ float with_rest(float sum, float rest) { return fabsf(sum) <= 3.402823466e38f ? sum + rest : sum; }

__device__ int64_t place(const CacheSide& s, uint32_t block, uint32_t at) { return (int64_t)((uint64_t)block * s.block + at * s.token); }
__device__ int64_t scale_place(const CacheSide& s, uint32_t block, uint32_t at) {
    return (int64_t)((uint64_t)block * s.scale_block + at * s.scale_token);
}

// ---- wide -------------------------------------------------------------------------------------

// Which rows a workgroup has: tile `tile` of all the sequences' tiles of ROWS rows.
struct Tile {
    uint32_t seq, first_token, tokens, first_row;
    int64_t len;              // of the sequence's keys, as given: loaded beside the starts, not behind them
    bool found;
};

template <uint32_t ROWS>
__device__ Tile find_tile(const AttentionArgs& a, const WideWalk& w, uint32_t tile) {
    Tile t{0, 0, 0, 0, 0, false};
    if (w.starts == nullptr) {
        t.tokens = a.n_rows;
        t.first_row = tile * ROWS;
        t.len = w.lens[0];
        t.found = t.first_row < t.tokens * a.group;
        return t;
    }
    const uint32_t lane = threadIdx.x % 64u;
    uint32_t before = 0;
    for (uint32_t base = 0; base < w.n_seqs; base += 64u) {       // 64 sequences at a time, by every wave alike
        const uint32_t b = base + lane;
        int64_t first = 0, last = 0, len = 0;
        if (b < w.n_seqs) {
            first = w.starts[b];
            last = w.starts[b + 1];
            len = w.lens[b];
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
            t.len = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)((uint64_t)len >> 32), at) << 32 |
                              (uint32_t)__builtin_amdgcn_readlane((uint32_t)len, at));
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

// out = V^T P^T / l with P = exp2(S - m), S = K Q^T * scale * log2 e, over tiles of KEYS keys: bound by the matrix units, with the
// exponentials, the maximum and the widening of e4m3 on the vector units next to them. 256 rows per workgroup, so that a tile
// put into LDS once serves eight waves, and two waves per SIMD, so that one has the matrix unit while the other has the vector
// unit. Measured: a causal prompt of 8192 tokens, 32 heads over 8 of 128 in bf16, 563 to 575 us, 960 to 980 TFLOP/s (matrix units busy 41 %
// of the cycles; a large matrix product reaches 1560 to 1580); 250 tokens behind 16000 in e4m3 81 us in a long series of launches, 90 in its
// first twenty. Without the turns, four waves of 32 rows: 1399 us. Heads of 64: 610 TFLOP/s, as the exponentials weigh twice. Heads of 256
// take tiles of 32 keys, since LDS holds no more, and spill about 58 registers: 330 TFLOP/s (211 for 4096 tokens, 16 heads over 4).
// The weights go into the second product rounded to T: an output's error against 64 bits is 2.1e-3 of the outputs' size in bf16 then, 1.6e-3
// being the output's own rounding (2.2e-4 and 1.9e-4 in fp16). Their rest as a second operand (see rest8) would take that away and cost the
// matrix units half as much again: 770 us instead of 574 for the causal prompt, 109 instead of 86.5 for the e4m3 chunk and its join.
template <typename T, bool FP8, int DP, int KEYS>
__global__ __launch_bounds__(kWideThreads, 2) void wide_attention_kernel(const AttentionArgs a, const WideWalk w) {
    constexpr uint32_t kRows = hfk::kWideRows, kThreads = kWideThreads, kWaves = kThreads / 64;
    constexpr uint32_t kPieces = FP8 ? DP / 16 : DP / 8;                  // 16-byte pieces of a cached row
    constexpr uint32_t kLoads = (KEYS * kPieces + kThreads - 1) / kThreads;
    constexpr uint32_t kKeyStage = KEYS * kKeyRow<DP>, kValueStage = KEYS * kValueRow<DP>;
    constexpr uint32_t kRing = 8;                                         // tiles whose places are kept
    __shared__ __align__(16) char k_lds[3 * kKeyStage];
    __shared__ __align__(16) char v_lds[3 * kValueStage];
    __shared__ TileKeys<KEYS> keys[kRing];
    __shared__ TileScales<FP8 ? KEYS : 1> scales[kRing];
    __shared__ uint32_t not_finite[2];                                    // first and last tile that values were taken out of

    const uint32_t tid = threadIdx.x, lane = tid % 64u, wave = __builtin_amdgcn_readfirstlane(tid / 64u), col = lane % 32u, half = lane / 32u;
    const uint32_t head = blockIdx.x % a.cache_heads, rest = blockIdx.x / a.cache_heads;
    const uint32_t split = rest % w.splits;
    const Tile t = find_tile<kRows>(a, w, w.tiles - 1u - rest / w.splits);   // long tiles of a causal walk first
    if (!t.found) return;

    const uint32_t n_tile_rows = t.tokens * a.group;
    const uint32_t len = clamp_len(t.len, w.width, a.split.T);
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
        // (the builtin gives an int: a half that begins with a one must not be extended by its sign)
        const uint32_t high = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)), low = __builtin_amdgcn_readfirstlane((uint32_t)x);
        return (uint64_t)high << 32 | low;
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
        if (found) {
            atomicMin(&not_finite[0], tile);
            atomicMax(&not_finite[1], tile);
        }
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
    constexpr float kLift = kLiftOf<T>;
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
    const auto weigh = [&] {
        const float base = top == kMinusInf ? 0.0f : top * a.score_scale - kLift;
        float add = 0.0f;
        for (int b = 0; b < KEYS / 32; ++b)
            for (int h = 0; h < 2; ++h) {
                float e[8];
                for (int i = 0; i < 8; ++i) {
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x.s[b][8 * h + i], a.score_scale, -base));
                    add += e[i];
                }
                y.p[2 * b + h] = pack8<T>(e);
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
    if (tid == 0) {
        not_finite[0] = ~0u;
        not_finite[1] = 0u;
    }
    if (n_tiles == 1) {      // nothing to overlap with, and nothing to load ahead: a short prompt's latency
        if (wave == 0) put_keys(0, load_entry(0));
        __syncthreads();
        const uint64_t seen = as_scalar(keys[0].seen);
        read_k_places(0);
        read_v_places(0);
        load_k(k_reg);
        load_v();
        store_k(0, k_reg);
        store_v(0, seen);
        __syncthreads();
        if (any_row) {
            first_product(0);
            hide(0, seen);
            raise();
            read_ahead(0);
            weigh();
            second_product(0);
        }
    } else if (n_tiles != 0) {
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
    // All scores NaN: no maximum was found, but something was seen, and the sums say what.
    if (top == kMinusInf && total != total) top = 0.0f;
    const uint64_t heads = a.cache_heads * a.group;
    if (owns) {
        const uint64_t place = (uint64_t)token * heads + q_head;
        const float high = top == kMinusInf ? kMinusInf : top * a.score_scale - kLift;
        if (w.to.sum != nullptr) {
            const uint64_t at = (uint64_t)split * a.n_rows * heads + place;
            if (half == 0) {
                w.to.stat[2 * at] = high;
                w.to.stat[2 * at + 1] = total;
            }
            if (top != kMinusInf) {
                float* dst = w.to.sum + at * a.dim;
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

    // Rare and slow: what was taken out of V, to every row that sees the key it belongs to. Sums of values that are no
    // numbers do not change when one of them comes twice, so that tiles between these that nothing was taken out of do no harm.
    __syncthreads();
    if (n_tiles == 0 || not_finite[0] == ~0u) return;
    const uint32_t from_key = first_key + not_finite[0] * KEYS, past = first_key + (not_finite[1] + 1u) * KEYS;
    for (uint32_t n = tid; n < kRows * a.dim; n += kThreads) {
        const uint32_t r = t.first_row + n / a.dim, d = n % a.dim;
        if (r >= n_tile_rows) break;
        const uint32_t of = r / a.group, of_head = head * a.group + r % a.group;
        uint32_t until = (uint32_t)seen_by(of) < end_key ? (uint32_t)seen_by(of) : end_key;
        until = until < past ? until : past;
        float add = 0.0f;
        for (uint32_t key = from_key; key < until; ++key) {
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
        if (w.to.sum != nullptr) {
            w.to.sum[((uint64_t)split * a.n_rows * heads + at_token * heads + of_head) * a.dim + d] += add;
        } else {
            uint16_t& to = reinterpret_cast<uint16_t*>(a.out + (int64_t)at_token * a.out_token + (int64_t)of_head * a.out_head)[d];
            to = (uint16_t)T::pack2(T::to_float(to) + add, 0.0f);
        }
    }
}

// ---- narrow -----------------------------------------------------------------------------------

__device__ uint32_t units_of(const NarrowWalk& w, uint32_t T, uint32_t seq) {
    return (clamp_len(w.lens[seq], w.width, T) + w.unit - 1u) / w.unit;
}

// Units of all sequences, and of those before `seq`. By every wave alike, 64 sequences at a time.
struct UnitSums {
    uint32_t all, before;
};
__device__ UnitSums sum_units(const NarrowWalk& w, uint32_t T, uint32_t seq) {
    const uint32_t lane = threadIdx.x % 64u;
    uint32_t all = 0, before = 0;
    for (uint32_t b = lane; b < w.n_seqs; b += 64u) {
        const uint32_t n = units_of(w, T, b);
        all += n;
        before += b < seq ? n : 0u;
    }
    for (uint32_t o = 32; o != 0; o >>= 1) {
        all += __shfl_xor(all, (int)o);
        before += __shfl_xor(before, (int)o);
    }
    return {(uint32_t)__builtin_amdgcn_readfirstlane(all), (uint32_t)__builtin_amdgcn_readfirstlane(before)};
}
__device__ uint32_t share_of(const NarrowWalk& w, uint32_t all) {
    const uint32_t n = (all + w.ranges - 1u) / w.ranges;
    return n == 0 ? 1u : n;
}

// The sequence that unit `unit` is in, its first unit and its length. There is one: unit < all.
struct UnitPlace {
    uint32_t seq, start, len;
};
// `lens` of 64 sequences from `base` on, a lane each; `before`: the units of those before them.
__device__ bool find_unit_in(const NarrowWalk& w, uint32_t len, uint32_t base, uint32_t unit, uint32_t& before, UnitPlace& found) {
    const uint32_t lane = threadIdx.x % 64u, mine = (len + w.unit - 1u) / w.unit;
    uint32_t upto = mine;
    for (uint32_t o = 1; o < 64u; o <<= 1) {
        const uint32_t other = __shfl_up(upto, o);
        if (lane >= o) upto += other;
    }
    const uint64_t past = __ballot(before + upto > unit);
    if (past != 0) {
        const int at = __builtin_ctzll(past);
        found = {base + at, before + (uint32_t)__builtin_amdgcn_readlane(upto, at) - (uint32_t)__builtin_amdgcn_readlane(mine, at),
                 (uint32_t)__builtin_amdgcn_readlane(len, at)};
        return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    return false;
}

// The units of range `range`: [first, end), and where the first lies. false: there are none.
__device__ bool find_range(const NarrowWalk& w, uint32_t T, uint32_t range, uint32_t& first, uint32_t& end, UnitPlace& found) {
    const uint32_t lane = threadIdx.x % 64u;
    uint32_t len = lane < w.n_seqs ? clamp_len(w.lens[lane], w.width, T) : 0u, all = (len + w.unit - 1u) / w.unit;
    for (uint32_t b = lane + 64u; b < w.n_seqs; b += 64u) all += units_of(w, T, b);
    for (uint32_t o = 32; o != 0; o >>= 1) all += __shfl_xor(all, (int)o);
    all = __builtin_amdgcn_readfirstlane(all);
    const uint32_t share = share_of(w, all);
    if ((uint64_t)range * share >= all) return false;
    first = range * share;
    end = all - first < share ? all : first + share;
    uint32_t before = 0;
    for (uint32_t base = 0; base < w.n_seqs; base += 64u) {
        if (base != 0) len = base + lane < w.n_seqs ? clamp_len(w.lens[base + lane], w.width, T) : 0u;
        if (find_unit_in(w, len, base, first, before, found)) return true;
    }
    return false;
}

// The same sums for 16 * R rows of a cache head: few rows per key, bound by reading the cache. Each wave has keys of its own,
// 32 at a time, and meets no barrier on the way; all sequences' keys are one row that the resident workgroups share
// equally, since rounds of more workgroups, one for each sequence and a fixed number of its keys, ended ragged (24 sequences of 5 to 8000
// tokens in e4m3, 64 heads over 8 of 128: 71 us and 7 for the join, 4.4 TB/s in all; 184 us in such rounds). bf16 caches are read
// at 5.2 to 5.5 TB/s, a long copy moves 5.16 and a long read 6.1.
// HEADS == 4: a wave for each of four neighbouring cache heads, all at the same keys. HEADS == 1: four waves at one head, whose
// sums meet in LDS.
template <typename T, bool FP8, int DP, int R, int HEADS>
__global__ __launch_bounds__(256, R * DP <= 256 && DP != 256 ? 2 : 1) void narrow_attention_kernel(const AttentionArgs a, const NarrowWalk prefix, const NarrowWalk own) {
    constexpr int kKSteps = DP / 32;        // matrix instructions of the first product
    constexpr int kCols = DP / 16;          // values of V per lane and key
    constexpr uint32_t kRegs = R * kCols * 4, kWavesPerHead = 4 / HEADS, kUnit = kWavesPerHead * 32;
    // The weights' rest (see rest8) where the kernel waits for memory and has registers to spare: 83.2 us without and with it
    // for the decoding step of 24 sequences, 11.5 and 11.9 for one sequence, whose errors then are the output's own rounding.
    constexpr bool kRest = R * DP <= 128;
    constexpr int kRowPieces = FP8 ? DP / 16 : DP / 8;                   // 16-byte pieces of a cached row
    constexpr uint32_t kRowBytes = kRowPieces * 16 + 16;                 // of K in LDS: 16 rows' pieces of one column, no bank twice
    struct alignas(16) WaveLds {                                         // a wave's own: no barrier, LDS serves a wave in order
        char k[32 * kRowBytes];
        int64_t place[32][2];                                            // of a key's K and V
        float scale[2][FP8 ? 32 : 1];
    };
    static_assert(alignof(WaveLds) == 16 && sizeof(WaveLds) % 16 == 0);  // every wave's K is written and read 16 bytes at a time
    __shared__ float tops[4][R * 16], sums[4][R * 16];
    __shared__ __align__(16) union {
        WaveLds wave[4];
        float o[2][HEADS == 1 ? kRegs * 64 : 1];                         // once the keys are done
    } lds;

    const uint32_t tid = threadIdx.x, lane = tid % 64u, wave = __builtin_amdgcn_readfirstlane(tid / 64u), col = lane % 16u, quarter = lane / 16u;
    const bool is_prefix = blockIdx.x < prefix.groups;
    const NarrowWalk& w = is_prefix ? prefix : own;
    const uint32_t group_id = is_prefix ? blockIdx.x : blockIdx.x - prefix.groups;
    // Workgroups go to the XCDs in turn. Where there are ranges for each, all heads of the same keys go to one: where tokens are
    // stored whole its L2 then takes whole lines and pages, and the scales' lines once.
    const uint32_t head_groups = a.cache_heads / HEADS, same_keys = head_groups * w.tiles;
    const bool by_xcd = w.ranges % 8u == 0;
    const uint32_t of_range = by_xcd ? group_id / 8u % same_keys : group_id % same_keys;
    const uint32_t range = by_xcd ? group_id / 8u / same_keys * 8u + group_id % 8u : group_id / same_keys;
    const uint32_t head = of_range % head_groups * HEADS + wave / kWavesPerHead, tile = of_range / head_groups;
    const uint32_t key_wave = wave % kWavesPerHead;

    const uint32_t T_block = a.split.T;
    uint32_t unit = 0, end_unit = 0;
    UnitPlace at_seq{};
    if (!find_range(w, T_block, range, unit, end_unit, at_seq)) return;
    // One part of the range after the other: keys [first_key, end_key) of sequence `seq`.
    for (uint32_t seq = at_seq.seq, start_unit = at_seq.start; unit < end_unit && seq < w.n_seqs; ++seq) {
        const uint32_t len = seq == at_seq.seq ? at_seq.len : clamp_len(w.lens[seq], w.width, T_block), n_units = (len + w.unit - 1u) / w.unit;
        const uint32_t stop = start_unit + n_units < end_unit ? start_unit + n_units : end_unit;
        if (n_units == 0) continue;
        const uint32_t first_key = (unit - start_unit) * kUnit;
        const uint32_t end_key = (stop - start_unit) * kUnit < len ? (stop - start_unit) * kUnit : len;
        unit = stop;
        start_unit += n_units;
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
                // an e4m3 row is read 16 values at a time, which two steps share
                const uint32_t d = FP8 ? (s / 2) * 64u + quarter * 16u + (s % 2) * 8u : s * 32u + quarter * 8u;
                u32x4 x{0, 0, 0, 0};
                if (owns[r] && d < a.dim) x = *reinterpret_cast<const u32x4*>(src + 2u * d);
                q[r][s] = as_vec8<T>(x);
            }
        }
        f32x4 o[R][kCols], o_rest[kRest ? R : 1][kRest ? kCols : 1];
        float top[R], sum[R];
        for (int r = 0; r < R; ++r) {
            top[r] = kMinusInf;
            sum[r] = 0.0f;
            for (int c = 0; c < kCols; ++c) {
                o[r][c] = f32x4{0, 0, 0, 0};
                if constexpr (kRest) o_rest[r][c] = f32x4{0, 0, 0, 0};
            }
        }

        const int64_t* table = w.table + (uint64_t)seq * w.width;
        const char* k_base = a.k.values + (int64_t)head * a.k.head;
        const char* v_base = a.v.values + (int64_t)head * a.v.head;
        const float* k_scale_base = FP8 ? a.k.scales + (int64_t)head * a.k.scale_head : nullptr;
        const float* v_scale_base = FP8 ? a.v.scales + (int64_t)head * a.v.scale_head : nullptr;
        // A tile of 32 keys. Lane l looks up key l % 32 and, of an e4m3 cache, loads one scale: K's in the lower half, V's in the
        // upper. A key that is not visible is given the cache's first token: its score is masked and its values are taken for
        // zeros. Rows are loaded whole by neighbouring lanes, 16 bytes each where they can be: four neighbours then make one
        // request of 64 bytes, where a lane for each key would make four. K goes through LDS into the first product's order. (24
        // sequences of 8000 tokens, 8 heads of 128 in e4m3: 98 us; K loaded in the first product's order 104 us.)
        const uint32_t last_entry = w.width == 0 ? 0u : w.width - 1u;
        WaveLds& mine = lds.wave[wave];
        const auto look_up = [&](uint32_t key0) -> int64_t {
            const uint32_t n = a.split.block32(key0 + lane % 32u);
            return table[n < last_entry ? n : last_entry];
        };
        constexpr int kWords = FP8 ? kCols / 4 : kCols / 2;              // of V per lane and key
        constexpr int kRowsAtOnce = 64 / kRowPieces, kLoads = 32 / kRowsAtOnce;
        const uint32_t piece = lane % kRowPieces, piece_row = lane / kRowPieces;
        const bool piece_exists = piece * (FP8 ? 16u : 8u) < a.dim;
        const uint32_t d0 = col * kCols < a.dim ? col * kCols : 0u;      // columns that do not exist are computed for nothing
        constexpr float kLift = kLiftOf<T>;
        const float lazily = kLazily / a.score_scale;
        struct Tile32 {
            u32x4 k[kLoads];
            uint32_t v[8][kWords];
            float scale;
            uint32_t seen;
        };
        const auto load_tile = [&](uint32_t key0, int64_t entry) -> Tile32 {
            Tile32 x;
            const uint32_t key = key0 + lane % 32u;
            const bool ok = key < end_key && (uint64_t)entry < a.blocks;
            x.seen = (uint32_t)__ballot(ok);
            const uint32_t block = ok ? (uint32_t)entry : 0u, at = ok ? key - a.split.block32(key) * a.split.T : 0u;
            // (a scale of a key that is not visible may be anything, and one that is no number makes NaN even of a zero)
            if constexpr (FP8) {
                const float scale = lane < 32u ? k_scale_base[scale_place(a.k, block, at)] : v_scale_base[scale_place(a.v, block, at)];
                x.scale = ok ? scale : 1.0f;
            }
            mine.place[lane % 32u][lane / 32u] = lane < 32u ? place(a.k, block, at) : place(a.v, block, at);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int n = 0; n < kLoads; ++n) {
                x.k[n] = u32x4{0, 0, 0, 0};
                const int64_t from = mine.place[n * kRowsAtOnce + piece_row][0];
                x.k[n] = *reinterpret_cast<const u32x4*>(k_base + from + (piece_exists ? piece * 16u : 0u));
            }
            // Value j of this quarter is key 16 (j / 4) + 4 quarter + j % 4, in the order in which the first product leaves its
            // scores; this lane has columns col * kCols ..+kCols-1 of all eight.
            for (int j = 0; j < 8; ++j) {
                const char* src = v_base + mine.place[j / 4 * 16 + quarter * 4 + j % 4][1] + d0 * (FP8 ? 1u : 2u);
                uint32_t* to = x.v[j];
                if constexpr (kWords == 1) {
                    to[0] = *reinterpret_cast<const uint32_t*>(src);
                } else if constexpr (kWords == 2) {
                    const u32x2 y = *reinterpret_cast<const u32x2*>(src);
                    to[0] = y[0];
                    to[1] = y[1];
                } else {
                    for (int n = 0; n < kWords / 4; ++n) {
                        const u32x4 y = *reinterpret_cast<const u32x4*>(src + 16 * n);
                        for (int i = 0; i < 4; ++i) to[4 * n + i] = y[i];
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            return x;
        };
        const auto compute = [&](Tile32& now) {
            const uint32_t seen = now.seen;
            for (int n = 0; n < kLoads; ++n)
                *reinterpret_cast<u32x4*>(mine.k + (n * kRowsAtOnce + piece_row) * kRowBytes + piece * 16u) = piece_exists ? now.k[n] : u32x4{0, 0, 0, 0};
            if constexpr (FP8) mine.scale[lane / 32u][lane % 32u] = now.scale;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            float k_scale[2], v_scale[8];
            if constexpr (FP8) {
                for (int t = 0; t < 2; ++t) {
                    k_scale[t] = mine.scale[0][t * 16 + col];
                    const f32x4 y = *reinterpret_cast<const f32x4*>(&mine.scale[1][t * 16 + quarter * 4]);
                    for (int j = 0; j < 4; ++j) v_scale[4 * t + j] = y[j];
                }
            }
            if (seen != 0xffffffffu)
                for (int j = 0; j < 8; ++j)
                    if (((seen >> (j / 4 * 16u + quarter * 4u + j % 4)) & 1u) == 0)
                        for (int x = 0; x < kWords; ++x) now.v[j][x] = 0u;

            f32x4 s[R][2];
            for (int r = 0; r < R; ++r)
                for (int t = 0; t < 2; ++t) s[r][t] = f32x4{0, 0, 0, 0};
            for (int t = 0; t < 2; ++t) {
                u32x4 raw[kRowPieces / 4];
                for (int n = 0; n < kRowPieces / 4; ++n)
                    raw[n] = *reinterpret_cast<const u32x4*>(mine.k + (t * 16 + col) * kRowBytes + (n * 4 + quarter) * 16u);
                for (int n = 0; n < kKSteps; ++n) {
                    u32x4 x;
                    if constexpr (FP8) {
                        const uint32_t w0 = raw[n / 2][2 * (n % 2)], w1 = raw[n / 2][2 * (n % 2) + 1];
                        x = u32x4{T::template from_fp8<false>(w0, k_scale[t]), T::template from_fp8<true>(w0, k_scale[t]),
                                  T::template from_fp8<false>(w1, k_scale[t]), T::template from_fp8<true>(w1, k_scale[t])};
                    } else {
                        x = raw[n];
                    }
                    for (int r = 0; r < R; ++r) s[r][t] = T::mfma16(as_vec8<T>(x), q[r][n], s[r][t]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (seen != 0xffffffffu)
                for (int r = 0; r < R; ++r)
                    for (int t = 0; t < 2; ++t)
                        for (int i = 0; i < 4; ++i)
                            if (((seen >> (t * 16u + quarter * 4u + i)) & 1u) == 0) s[r][t][i] = kMinusInf;

            typename T::Vec8 p[R], rest[kRest ? R : 1];
            for (int r = 0; r < R; ++r) {
                float high = kMinusInf;
                for (int t = 0; t < 2; ++t)
                    for (int i = 0; i < 4; ++i) high = fmaxf(high, s[r][t][i]);
                high = max_across_32(max_across_16(high));
                if (__any(high > top[r] + lazily)) {
                    const float now = fmaxf(top[r], high);
                    const float keep = now == kMinusInf ? 1.0f : __builtin_amdgcn_exp2f((top[r] - now) * a.score_scale);
                    top[r] = now;
                    sum[r] *= keep;
                    for (int c = 0; c < kCols; ++c) {
                        o[r][c] *= keep;
                        if constexpr (kRest) o_rest[r][c] *= keep;
                    }
                }
                const float base = top[r] == kMinusInf ? 0.0f : top[r] * a.score_scale - kLift;
                float e[8], add = 0.0f;
                for (int t = 0; t < 2; ++t)
                    for (int i = 0; i < 4; ++i) {
                        e[4 * t + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][t][i], a.score_scale, -base));
                        add += e[4 * t + i];
                    }
                sum[r] += add;
                p[r] = pack8<T>(e);
                if constexpr (kRest) rest[r] = rest8<T>(e, p[r]);
            }
            // Columns 2 w and 2 w + 1 of eight keys out of eight dwords.
            for (int x = 0; x < kCols / 2; ++x) {
                uint32_t two[8];
                for (int j = 0; j < 8; ++j) {
                    if constexpr (FP8) two[j] = x % 2 ? T::template from_fp8<true>(now.v[j][x / 2], v_scale[j]) : T::template from_fp8<false>(now.v[j][x / 2], v_scale[j]);
                    else two[j] = now.v[j][x];
                }
                u32x4 even, odd;
                for (int i = 0; i < 4; ++i) {
                    even[i] = __builtin_amdgcn_perm(two[2 * i + 1], two[2 * i], 0x05040100u);
                    odd[i] = __builtin_amdgcn_perm(two[2 * i + 1], two[2 * i], 0x07060302u);
                }
                for (int r = 0; r < R; ++r) {
                    o[r][2 * x] = T::mfma16(as_vec8<T>(even), p[r], o[r][2 * x]);
                    o[r][2 * x + 1] = T::mfma16(as_vec8<T>(odd), p[r], o[r][2 * x + 1]);
                    if constexpr (kRest) {
                        o_rest[r][2 * x] = T::mfma16(as_vec8<T>(even), rest[r], o_rest[r][2 * x]);
                        o_rest[r][2 * x + 1] = T::mfma16(as_vec8<T>(odd), rest[r], o_rest[r][2 * x + 1]);
                    }
                }
            }
        };
        const uint32_t start = first_key + key_wave * 32u;
        if (start < end_key) {
            int64_t ahead = look_up(start);      // a tile early; loading the tile itself early was no faster: its registers cost waves
            for (uint32_t key0 = start; key0 < end_key; key0 += kUnit) {
                Tile32 now = load_tile(key0, ahead);
                ahead = look_up(key0 + kUnit);
                compute(now);
            }
        }

        for (int r = 0; r < R; ++r) {
            sum[r] = sum_across_32(sum_across_16(sum[r]));
            // All scores NaN: no maximum was found, but something was seen, and the sums say what.
            if (top[r] == kMinusInf && sum[r] != sum[r]) top[r] = 0.0f;
            if constexpr (kRest)
                for (int c = 0; c < kCols; ++c)
                    for (int i = 0; i < 4; ++i) o[r][c][i] = with_rest(o[r][c][i], o_rest[r][c][i]);
        }
        if constexpr (HEADS == 1) {      // the four waves' sums into wave 0's
            for (int r = 0; r < R; ++r) {
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
                            for (int i = 0; i < 4; ++i) lds.o[wave - step][((r * kCols + c) * 4 + i) * 64 + lane] = o[r][c][i];
                __syncthreads();
                if (wave < step)
                    for (int r = 0; r < R; ++r)
                        for (int c = 0; c < kCols; ++c)
                            for (int i = 0; i < 4; ++i) o[r][c][i] += lds.o[wave][((r * kCols + c) * 4 + i) * 64 + lane];
                __syncthreads();
            }
        }
        if (key_wave == 0)
            for (int r = 0; r < R; ++r) {
                if (!owns[r]) continue;
                const uint64_t heads = a.cache_heads * a.group;
                const uint64_t at = w.n_seqs == 1 ? (uint64_t)range * a.n_rows * heads + token[r] * heads + q_head[r] : ((uint64_t)range + seq) * heads + q_head[r];
                if (quarter == 0) {
                    w.to.stat[2 * at] = top[r] == kMinusInf ? kMinusInf : top[r] * a.score_scale - kLift;
                    w.to.stat[2 * at + 1] = sum[r];
                }
                if (top[r] == kMinusInf) continue;
                for (int i = 0; i < 4; ++i) {
                    const uint32_t d = (quarter * 4u + i) * kCols;
                    if (d >= a.dim) continue;
                    for (int c = 0; c < kCols; c += 4)
                        *reinterpret_cast<f32x4*>(w.to.sum + at * a.dim + d + c) = f32x4{o[r][c][i], o[r][c + 1][i], o[r][c + 2][i], o[r][c + 3][i]};
                }
            }
    }
}

// ---- join -------------------------------------------------------------------------------------

struct Join {
    Partials shared;          // splits that have every row: of a wide launch, or of a narrow one over a prefix
    uint32_t shared_splits;   // of a wide launch; 0: as many of prefix's ranges as its length takes
    NarrowWalk prefix, own;   // own.n_seqs == 0: no splits of the rows' own sequences
    const int64_t* starts;    // of prompts: rows of no sequence have no splits and stay as they are
    uint32_t n_seqs;
};

// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s over the splits s of a row, bound by reading them where rows are many (2048
// rows of 34 splits of 128 values, 36 MB: 10.4 us, 3.4 TB/s) and by the chain lengths, statistics, sums where they are few (5 us).
// The splits' sums of a query row, each brought to the common maximum, by WAVES waves of a workgroup: one for many rows, four
// where rows are few and their splits many.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void join_splits_kernel(const AttentionArgs a, const Join j) {
    __shared__ f32x4 sums[WAVES][WAVES > 1 ? 64 : 1];
    __shared__ float totals[WAVES], highs[WAVES];
    const uint32_t lane = threadIdx.x % 64u, heads = a.cache_heads * a.group, wave = threadIdx.x / 64u % WAVES;
    const uint64_t rows = (uint64_t)a.n_rows * heads;
    const uint64_t row = (uint64_t)blockIdx.x * (4u / WAVES) + threadIdx.x / (64u * WAVES);
    if (row >= rows) return;      // all waves of the row
    const uint32_t token = __builtin_amdgcn_readfirstlane((uint32_t)(row / heads)), head = (uint32_t)(row % heads);
    if (j.starts != nullptr) {
        bool inside = false;
        for (uint32_t b = lane; b < j.n_seqs; b += 64u) {
            const int64_t first = j.starts[b], last = j.starts[b + 1];
            inside |= first >= 0 && last <= (int64_t)a.n_rows && (int64_t)token >= first && (int64_t)token < last;
        }
        if (!__any(inside)) return;
    }
    // The splits there are: first those that have every row, then the parts of this row's own sequence.
    uint32_t n_shared = j.shared_splits, n_own = 0;
    if (j.prefix.n_seqs != 0) {
        const uint32_t all = units_of(j.prefix, a.split.T, 0), share = share_of(j.prefix, all);
        n_shared = (all + share - 1u) / share;
    }
    uint64_t own_at = 0;
    if (j.own.n_seqs == 1) {
        const uint32_t all = units_of(j.own, a.split.T, 0), share = share_of(j.own, all);
        n_own = (all + share - 1u) / share;
        own_at = head;
    } else if (j.own.n_seqs != 0) {
        const UnitSums u = sum_units(j.own, a.split.T, token);
        const uint32_t mine = units_of(j.own, a.split.T, token), share = share_of(j.own, u.all);
        if (mine != 0) {
            const uint32_t first = u.before / share;
            n_own = (u.before + mine - 1u) / share - first + 1u;
            own_at = ((uint64_t)first + token) * heads + head;
        }
    }
    const uint32_t splits = n_shared + n_own;
    // Place of split s, in rows; of the second kind the next split is `heads` rows further.
    const auto place_of = [&](uint32_t s) -> uint64_t { return s < n_shared ? s * rows + row : own_at + (uint64_t)(s - n_shared) * heads; };
    const auto stat_of = [&](uint32_t s) -> const float* { return (s < n_shared ? j.shared.stat : j.own.to.stat) + 2 * place_of(s); };

    // A row of one split takes `lanes` lanes of four values; the wave reads 64 / lanes splits at a time.
    const uint32_t lanes = a.dim <= 64u ? 16u : a.dim <= 128u ? 32u : 64u, side_by_side = 64u / lanes;
    const uint32_t d = lane % lanes * 4u, mine = lane / lanes;
    // One pass: 64 splits' statistics at a time, a running maximum, and four loads of sums in flight that wait for no weight. A
    // split that saw nothing has no sum written: what lies there is read and not used, as its weight kUnseen says. A weight that is
    // zero in 32 bits only still multiplies: NaN among a split's sums stays NaN whatever the other splits hold.
    constexpr float kUnseen = -1.0f;
    float high = kMinusInf, total = 0.0f;
    f32x4 acc{0, 0, 0, 0};
    for (uint32_t base = wave * 64u; base < splits; base += 64u * WAVES) {
        const uint32_t n = splits - base < 64u ? splits - base : 64u;
        float top = kMinusInf, sum = 0.0f;
        if (lane < n) {
            const float* stat = stat_of(base + lane);
            top = stat[0];
            sum = stat[1];
        }
        const auto load_sums = [&](uint32_t s, f32x4 (&x)[4]) {
            for (uint32_t i = 0; i < 4u; ++i) {
                const uint32_t from = base + s + i * side_by_side + mine;
                x[i] = f32x4{0, 0, 0, 0};
                if (from < splits && d < a.dim) x[i] = *reinterpret_cast<const f32x4*>((from < n_shared ? j.shared.sum : j.own.to.sum) + place_of(from) * a.dim + d);
            }
        };
        f32x4 x[4];
        load_sums(0, x);
        float most = top;
        for (uint32_t o = 32; o != 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, (int)o));
        if (most > high) {
            const float keep = __builtin_amdgcn_exp2f(high - most);      // 0 at first
            acc *= keep;
            total *= keep;
            high = most;
        }
        const float weight = top == kMinusInf ? kUnseen : __builtin_amdgcn_exp2f(top - high);
        total += weight == kUnseen ? 0.0f : weight * sum;
        for (uint32_t s = 0; s < n; s += 4u * side_by_side) {
            if (s != 0) load_sums(s, x);
            for (uint32_t i = 0; i < 4u; ++i) {
                const uint32_t from = s + i * side_by_side + mine;
                float by = __shfl(weight, (int)(from & 63u));              // by all lanes, whether they have such a split or not
                if (from >= n) by = kUnseen;
                for (int c = 0; c < 4; ++c) acc[c] += by == kUnseen ? 0.0f : by * x[i][c];
            }
        }
    }
    for (uint32_t o = lanes; o < 64u; o <<= 1)
        for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], (int)o);
    for (uint32_t o = 32; o != 0; o >>= 1) total += __shfl_xor(total, (int)o);
    if constexpr (WAVES > 1) {
        sums[wave][lane] = acc;
        if (lane == 0) {
            totals[wave] = total;
            highs[wave] = high;
        }
        __syncthreads();
        if (wave != 0) return;
        for (int x = 1; x < WAVES; ++x) high = fmaxf(high, highs[x]);
        acc = f32x4{0, 0, 0, 0};
        total = 0.0f;
        for (int x = 0; x < WAVES; ++x) {
            if (highs[x] == kMinusInf) continue;
            const float keep = __builtin_amdgcn_exp2f(highs[x] - high);
            acc += keep * sums[x][lane];
            total += keep * totals[x];
        }
    }
    const float inverse = high == kMinusInf ? 0.0f : 1.0f / total;
    if (d < a.dim && mine == 0) {
        char* dst = a.out + (int64_t)token * a.out_token + (int64_t)head * a.out_head + 2u * d;
        *reinterpret_cast<u32x2*>(dst) = u32x2{T::pack2(acc[0] * inverse, acc[1] * inverse), T::pack2(acc[2] * inverse, acc[3] * inverse)};
    }
    if (a.lse != nullptr && lane == 0) a.lse[row] = high == kMinusInf ? kMinusInf : (high + __log2f(total)) * kLn2;
}

// ---- host -------------------------------------------------------------------------------------

constexpr uint64_t kMostKeys = 1ull << 30;       // of one sequence

// Products of a block's stride, and of a token's inside its block, fit 32 bits.
bool block_fits(const hfk_cache_plane& p) {
    const uint64_t e = hfk::type_bytes(p.type), most = 0xffffffffull;
    const auto fits = [&](uint64_t block, uint64_t token) {      // by division: a product of the two passes 64 bits, too
        return (p.blocks <= 1 || block <= most) && (p.block_tokens == 1 || token <= most / (p.block_tokens - 1));
    };
    return fits(e * (uint64_t)p.block_stride, e * (uint64_t)p.token_stride) &&
           (p.type != HFK_FP8_E4M3 || fits((uint64_t)p.scale_block_stride, (uint64_t)p.scale_token_stride));
}

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
    if (!(a->scale >= 0x1p-100f && a->scale <= 0x1p100f)) return HFK_ERR_BAD_SIZE;      // kLazily / scale stays finite, too
    if (a->q_heads > 65535u || a->n_rows > 0x7fffffffull || a->n_rows * a->q_heads > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    if (!block_fits(k) || !block_fits(v)) return HFK_ERR_TOO_LARGE;
    if (!hfk::plane_aligned(k, 16) || !hfk::plane_aligned(v, 16) || !hfk::rows_aligned(a->q) || !hfk::rows_aligned(a->out))
        return HFK_ERR_BAD_ALIGNMENT;
    if (a->lse != nullptr && !hfk::multiple_of(a->lse, 4)) return HFK_ERR_BAD_ALIGNMENT;
    return HFK_OK;
}

CacheSide side_of(const hfk_cache_plane& p) {
    const int64_t e = hfk::type_bytes(p.type);
    const bool one = p.blocks <= 1;      // the stride of a single block means nothing
    return {static_cast<const char*>(p.values), p.type == HFK_FP8_E4M3 ? p.scales : nullptr, e * p.head_stride, p.scale_head_stride,
            one ? 0u : (uint32_t)(e * p.block_stride), (uint32_t)(e * p.token_stride), one ? 0u : (uint32_t)p.scale_block_stride,
            (uint32_t)p.scale_token_stride};
}

AttentionArgs fill(const hfk_attention* a) {
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
    return x;
}

// `rows` rows of sums and, behind them, of statistics; `at` moves behind both.
Partials take(char*& at, uint64_t rows, uint32_t dim) {
    Partials p{reinterpret_cast<float*>(at), reinterpret_cast<float*>(at + hfk::round_up(rows * dim * 4, 256))};
    at += hfk::partial_bytes(rows, dim);
    return p;
}

int check_workspace(void* workspace, uint64_t bytes, uint64_t needed) {
    if (needed == 0) return HFK_OK;
    if (workspace == nullptr) return HFK_ERR_NULL_POINTER;
    if (bytes < needed) return HFK_ERR_WORKSPACE_TOO_SMALL;
    return hfk::multiple_of(workspace, 256) ? HFK_OK : HFK_ERR_BAD_ALIGNMENT;
}

template <typename T, bool FP8>
void launch_wide(const AttentionArgs& x, const WideWalk& w, hipStream_t s) {
    switch (hfk::padded_head_dim(x.dim)) {
        case 64: wide_attention_kernel<T, FP8, 64, 64><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
        case 128: wide_attention_kernel<T, FP8, 128, 64><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
        default: wide_attention_kernel<T, FP8, 256, 32><<<w.groups, kWideThreads, 0, s>>>(x, w); break;
    }
}

template <typename T, bool FP8, int DP, int HEADS>
void launch_narrow_rows(const AttentionArgs& x, const NarrowWalk& prefix, const NarrowWalk& own, uint32_t row_blocks, hipStream_t s) {
    const uint32_t grid = prefix.groups + own.groups;
    if (row_blocks == 1) narrow_attention_kernel<T, FP8, DP, 1, HEADS><<<grid, 256, 0, s>>>(x, prefix, own);
    else if (row_blocks == 2) narrow_attention_kernel<T, FP8, DP, 2, HEADS><<<grid, 256, 0, s>>>(x, prefix, own);
    else if constexpr (DP != 256) narrow_attention_kernel<T, FP8, DP, 4, HEADS><<<grid, 256, 0, s>>>(x, prefix, own);
}

template <typename T, bool FP8, int DP>
void launch_narrow_heads(const AttentionArgs& x, const NarrowWalk& prefix, const NarrowWalk& own, uint32_t row_blocks, hipStream_t s) {
    if (hfk::narrow_heads(x.cache_heads) == 4) launch_narrow_rows<T, FP8, DP, 4>(x, prefix, own, row_blocks, s);
    else launch_narrow_rows<T, FP8, DP, 1>(x, prefix, own, row_blocks, s);
}

template <typename T, bool FP8>
void launch_narrow(const AttentionArgs& x, const NarrowWalk& prefix, const NarrowWalk& own, uint32_t row_blocks, hipStream_t s) {
    switch (hfk::padded_head_dim(x.dim)) {
        case 64: launch_narrow_heads<T, FP8, 64>(x, prefix, own, row_blocks, s); break;
        case 128: launch_narrow_heads<T, FP8, 128>(x, prefix, own, row_blocks, s); break;
        default: launch_narrow_heads<T, FP8, 256>(x, prefix, own, row_blocks, s); break;
    }
}

template <typename T>
void launch_join(const AttentionArgs& x, const Join& j, hipStream_t s) {
    const uint64_t rows = (uint64_t)x.n_rows * x.cache_heads * x.group;
    const uint64_t most = (uint64_t)j.shared_splits + j.prefix.ranges + j.own.ranges;      // of one row
    // 64 rows of 250 splits take 37 us with the attention before them by four waves, 56 by one; 1536 rows of 12 splits 8.2 and 7.2 us.
    if (most > 64 && rows <= 512) join_splits_kernel<T, 4><<<(uint32_t)rows, 256, 0, s>>>(x, j);
    else join_splits_kernel<T, 1><<<(uint32_t)((rows + 3) / 4), 256, 0, s>>>(x, j);
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
    *bytes = n_seqs == 0 || a->n_rows == 0 ? 0 : hfk::plan_prompt(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, n_seqs, keys).workspace;
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
    if (!hfk::launch_fits(p.wide.groups, kWideThreads)) return HFK_ERR_TOO_LARGE;
    const AttentionArgs x = fill(a);
    WideWalk w{};
    w.table = block_table;
    w.width = x.blocks != 0 ? (uint32_t)table_width : 0;      // a cache without blocks shows nothing
    w.starts = query_starts;
    w.lens = kv_lens;
    w.n_seqs = (uint32_t)n_seqs;
    w.causal = causal != 0;
    w.tiles = (uint32_t)p.wide.tiles;
    w.splits = p.wide.splits;
    w.groups = (uint32_t)p.wide.groups;
    char* at = static_cast<char*>(workspace);
    if (w.splits > 1) w.to = take(at, a->n_rows * a->q_heads * w.splits, x.dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(a, [&](auto type, auto fp8) {
        using T = decltype(type);
        launch_wide<T, decltype(fp8)::value>(x, w, s);
        if (w.splits > 1) {
            Join j{};
            j.shared = w.to;
            j.shared_splits = w.splits;
            j.starts = query_starts;
            j.n_seqs = w.n_seqs;
            launch_join<T>(x, j, s);
        }
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
    *bytes = a->n_rows == 0 ? 0 : hfk::plan_prefix(a->n_rows, a->q_heads, a->k.heads, a->k.head_dim, prefix, own).workspace;
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
    if (!hfk::launch_fits(p.wide.groups, kWideThreads) || !hfk::launch_fits(p.prefix.groups + p.own.groups, 256) ||
        !hfk::launch_fits(hfk::ceil_div(a->n_rows * a->q_heads, 4), 256) ||
        a->n_rows * hfk::ceil_div(own, hfk::narrow_unit(a->k.heads)) > 0x7fffffffull)
        return HFK_ERR_TOO_LARGE;
    const AttentionArgs x = fill(a);
    const bool narrow_prefix = prefix != 0 && !p.wide_prefix;
    char* at = static_cast<char*>(workspace);
    Join j{};
    WideWalk wide{};
    NarrowWalk none{};
    if (prefix != 0) j.shared = take(at, a->n_rows * a->q_heads * (p.wide_prefix ? p.wide.splits : p.prefix.ranges), x.dim);
    if (p.wide_prefix) {
        wide.table = prefix_blocks;
        wide.width = x.blocks != 0 ? (uint32_t)n_prefix_blocks : 0;      // a cache without blocks shows nothing
        wide.lens = prefix_len;
        wide.n_seqs = 1;
        wide.tiles = (uint32_t)p.wide.tiles;
        wide.splits = p.wide.splits;
        wide.groups = (uint32_t)p.wide.groups;
        wide.to = j.shared;
        j.shared_splits = wide.splits;
    }
    if (narrow_prefix) {
        j.prefix.table = prefix_blocks;
        j.prefix.width = x.blocks != 0 ? (uint32_t)n_prefix_blocks : 0;
        j.prefix.lens = prefix_len;
        j.prefix.n_seqs = 1;
        j.prefix.tokens_per_seq = (uint32_t)a->n_rows;
        j.prefix.tiles = (uint32_t)p.prefix.row_tiles;
        j.prefix.unit = hfk::narrow_unit(x.cache_heads);
        j.prefix.ranges = p.prefix.ranges;
        j.prefix.groups = (uint32_t)p.prefix.groups;
        j.prefix.to = j.shared;
    }
    j.own.table = block_table;
    j.own.width = x.blocks != 0 ? (uint32_t)table_width : 0;
    j.own.lens = kv_lens;
    j.own.n_seqs = (uint32_t)a->n_rows;
    j.own.tokens_per_seq = 1;
    j.own.tiles = (uint32_t)p.own.row_tiles;
    j.own.unit = hfk::narrow_unit(x.cache_heads);
    j.own.ranges = p.own.ranges;
    j.own.groups = (uint32_t)p.own.groups;
    j.own.to = take(at, hfk::own_splits(p.own, a->n_rows) * a->q_heads, x.dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(a, [&](auto type, auto fp8) {
        using T = decltype(type);
        constexpr bool kFp8 = decltype(fp8)::value;
        if (p.wide_prefix) launch_wide<T, kFp8>(x, wide, s);
        if (narrow_prefix && p.prefix.row_blocks == p.own.row_blocks) {
            launch_narrow<T, kFp8>(x, j.prefix, j.own, p.own.row_blocks, s);
        } else {
            if (narrow_prefix) launch_narrow<T, kFp8>(x, j.prefix, none, p.prefix.row_blocks, s);
            launch_narrow<T, kFp8>(x, none, j.own, p.own.row_blocks, s);
        }
        launch_join<T>(x, j, s);
    });
    return finish();
}

}  // extern "C"
