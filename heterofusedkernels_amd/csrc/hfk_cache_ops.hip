// Tokens into the paged cache and out of it: hfk_cache_write and hfk_cache_read of include/hfk.h.
//
// Both are one pass over the rows: a group of lanes takes one (token, head) row, 16 bytes of cached values per lane, and
// keeps it in registers between finding its largest value and writing it (write) or between loading and widening it
// (read). Keys and values go in one launch, so a decoding step pays one launch for both. What bounds
// a long call is HBM traffic, what bounds a short one is the launch. (8 heads of 128, keys and values: 16-bit caches 8192 tokens written in 12.0 us and
// read in 12.0, 5.6 TB/s; 32768 in 50.2 and 49.3, 5.4 TB/s; 1 to 1000 tokens in 4.8 to 4.9 us, which is the launch.)
#include <hip/hip_runtime.h>

#include <cstdint>

#include "hfk.h"
#include "hfk_cache_types.h"

namespace {

using hfk::BlockSplit;
using hfk::u32x2;
using hfk::u32x4;

constexpr uint32_t kMaxHeadDim = 1024;

struct Side {
    char* rows;               // tokens outside the cache
    char* values;             // the plane
    float* scales;
    int64_t row_token, row_head, block, token, head;      // strides, bytes
    int64_t scale_block, scale_token, scale_head;         // strides, floats
    BlockSplit heads;         // rows of a token
    uint32_t dim;
    uint32_t lanes;           // per row, a power of two
    uint32_t n_rows;          // tokens * heads
};

struct Args {
    Side side[2];
    const int64_t* slots;
    uint64_t capacity;        // slots of the cache
    BlockSplit split;
    uint32_t first_groups;    // workgroups of side 0; the rest are side 1's
};

// Where this lane's row lies; ok == false: no such row, or its slot is outside the cache.
struct Row {
    bool ok;
    char* outside;
    char* inside;
    float* scale;
    uint32_t lane;
};

__device__ Row locate(const Args& a, const Side& s, uint32_t group) {
    const uint32_t per_group = 256u / s.lanes;
    const uint64_t row = (uint64_t)group * per_group + threadIdx.x / s.lanes;
    Row r{};
    r.lane = threadIdx.x % s.lanes;
    if (row >= s.n_rows) return r;
    const uint32_t token = s.heads.block32((uint32_t)row), head = (uint32_t)row - token * s.heads.T;
    const uint64_t slot = (uint64_t)a.slots[token];      // a negative one is larger than any capacity
    if (slot >= a.capacity) return r;
    const uint64_t block = a.split.block(slot), at = slot - block * a.split.T;
    r.ok = true;
    r.outside = s.rows + (int64_t)token * s.row_token + (int64_t)head * s.row_head;
    r.inside = s.values + (int64_t)block * s.block + (int64_t)at * s.token + (int64_t)head * s.head;
    r.scale = s.scales == nullptr ? nullptr
                                  : s.scales + (int64_t)block * s.scale_block + (int64_t)at * s.scale_token + (int64_t)head * s.scale_head;
    return r;
}

__device__ const Side& side_of(const Args& a, uint32_t& group) {
    group = blockIdx.x;
    if (group < a.first_groups) return a.side[0];
    group -= a.first_groups;
    return a.side[1];
}

// ---- the scale of a row --------------------------------------------------------------------

// |x| where it is finite, else 0.
__device__ float finite_size(float x) {
    const float s = fabsf(x);
    return s <= 3.402823466e38f ? s : 0.0f;
}

__device__ float group_max(float x, uint32_t lanes) {
    for (uint32_t o = lanes >> 1; o != 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, (int)o));
    return x;
}

// Biased exponent of the smallest power of two s with most <= 448 * s. 448 = 1.75 * 2^8, so for most = m * 2^e that is
// 2^(e - 8), or twice that when m > 1.75.
__device__ uint32_t scale_exponent(float most) {
    const uint32_t bits = __float_as_uint(most);
    if (bits == 0) return 127u;                                       // 1.0
    const int32_t e = (int32_t)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(e < 1 ? 1 : e > 246 ? 246 : e);                 // 2^-126 .. 2^119
}

// x * 2^-k brought into e4m3's range: only an infinity, or a value next to fp32's own limit, lies outside. NaN passes.
__device__ float in_range(float x) {
    x = x > 448.0f ? 448.0f : x;
    return x < -448.0f ? -448.0f : x;
}

__device__ uint32_t four_fp8(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(in_range(a), in_range(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(in_range(c), in_range(d), p, true);
}

template <typename T>
__device__ void widen(u32x4 v, float (&x)[8]) {
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = T::to_float(v[i] & 0xffffu);
        x[2 * i + 1] = T::to_float(v[i] >> 16);
    }
}

// ---- write -----------------------------------------------------------------------------------

// CHUNKS pieces per lane: piece c of lane l is values (c * lanes + l) * PIECE ..+PIECE-1 of the row. PIECE is 8 for 16-bit
// caches, and 16 for e4m3 where everything is aligned for it: 16 bytes of the cache either way. (8192 tokens of 8 heads of 128,
// keys and values, from bf16 into e4m3: 12.1 us with 16 values, 4.2 TB/s; 14.5 with 8.)
template <typename T, bool FP8, int PIECE, int CHUNKS>
__global__ __launch_bounds__(256) void cache_write_kernel(const Args a) {
    constexpr int kLoads = PIECE / 8;
    uint32_t group;
    const Side& s = side_of(a, group);
    const Row r = locate(a, s, group);
    u32x4 v[CHUNKS][kLoads];
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t d = (c * s.lanes + r.lane) * PIECE;
        for (int n = 0; n < kLoads; ++n) {
            v[c][n] = u32x4{0, 0, 0, 0};
            if (r.ok && d < s.dim) v[c][n] = *reinterpret_cast<const u32x4*>(r.outside + 2 * d + 16 * n);
        }
    }
    if constexpr (!FP8) {
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t d = (c * s.lanes + r.lane) * PIECE;
            if (r.ok && d < s.dim) *reinterpret_cast<u32x4*>(r.inside + 2 * d) = v[c][0];
        }
    } else {
        float most = 0.0f;
        for (int c = 0; c < CHUNKS; ++c)
            for (int n = 0; n < kLoads; ++n) {
                float x[8];
                widen<T>(v[c][n], x);
                for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_size(x[i]));
            }
        const uint32_t e = scale_exponent(group_max(most, s.lanes));
        const float inverse = __uint_as_float((254u - e) << 23);
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t d = (c * s.lanes + r.lane) * PIECE;
            uint32_t p[PIECE / 4];
            for (int n = 0; n < kLoads; ++n) {
                float x[8];
                widen<T>(v[c][n], x);
                for (int i = 0; i < 8; ++i) x[i] *= inverse;
                p[2 * n] = four_fp8(x[0], x[1], x[2], x[3]);
                p[2 * n + 1] = four_fp8(x[4], x[5], x[6], x[7]);
            }
            if (!r.ok || d >= s.dim) continue;
            if constexpr (PIECE == 16) *reinterpret_cast<u32x4*>(r.inside + d) = u32x4{p[0], p[1], p[2], p[3]};
            else *reinterpret_cast<u32x2*>(r.inside + d) = u32x2{p[0], p[1]};
        }
        if (r.ok && r.lane == 0) *r.scale = __uint_as_float(e << 23);
    }
}

// Rows of any size, alignment and stride: one value at a time, the row read twice where it needs a scale. Bound by its requests, two bytes a
// lane: 8192 tokens of 8 heads of 128 from rows that lie two bytes beside a multiple of 16 in 29.4 us, into e4m3 in 48.7, where aligned rows
// take 12.0 and 11.9; read back in 29; up to 77 tokens the launch hides it (4.9 us either way). Heads of 100 values: 28.4 and 48.1 us.
template <typename T, bool FP8>
__global__ __launch_bounds__(256) void cache_write_any_kernel(const Args a) {
    uint32_t group;
    const Side& s = side_of(a, group);
    const Row r = locate(a, s, group);
    const uint16_t* in = reinterpret_cast<const uint16_t*>(r.outside);
    const uint32_t dim = r.ok ? s.dim : 0u;
    if constexpr (!FP8) {
        for (uint32_t d = r.lane; d < dim; d += s.lanes) reinterpret_cast<uint16_t*>(r.inside)[d] = in[d];
    } else {
        float most = 0.0f;
        for (uint32_t d = r.lane; d < dim; d += s.lanes) most = fmaxf(most, finite_size(T::to_float(in[d])));
        const uint32_t e = scale_exponent(group_max(most, s.lanes));
        const float inverse = __uint_as_float((254u - e) << 23);
        for (uint32_t d = r.lane; d < dim; d += s.lanes) {
            const float x = T::to_float(in[d]) * inverse;
            reinterpret_cast<uint8_t*>(r.inside)[d] = (uint8_t)four_fp8(x, 0.0f, 0.0f, 0.0f);
        }
        if (r.ok && r.lane == 0) *r.scale = __uint_as_float(e << 23);
    }
}

// ---- read ------------------------------------------------------------------------------------

// STREAM: the cache is read past the caches, which then keep more of the rows for whoever takes them next.
template <bool STREAM, typename V>
__device__ V load_cached(const char* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else return *reinterpret_cast<const V*>(p);
}

template <typename T, bool FP8, int PIECE, int CHUNKS, bool STREAM>
__global__ __launch_bounds__(256) void cache_read_kernel(const Args a) {
    constexpr int kWords = FP8 ? PIECE / 4 : PIECE / 2;      // of a piece in the cache
    uint32_t group;
    const Side& s = side_of(a, group);
    const Row r = locate(a, s, group);
    if (!r.ok) return;
    float scale = 1.0f;
    if constexpr (FP8) scale = *r.scale;
    uint32_t v[CHUNKS][kWords];
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t d = (c * s.lanes + r.lane) * PIECE;
        if (d >= s.dim) continue;
        if constexpr (kWords == 4) {
            const u32x4 x = load_cached<STREAM, u32x4>(r.inside + (FP8 ? d : 2 * d));
            for (int i = 0; i < 4; ++i) v[c][i] = x[i];
        } else {
            const u32x2 x = load_cached<STREAM, u32x2>(r.inside + d);
            v[c][0] = x[0];
            v[c][1] = x[1];
        }
    }
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t d = (c * s.lanes + r.lane) * PIECE;
        if (d >= s.dim) continue;
        if constexpr (!FP8) {
            *reinterpret_cast<u32x4*>(r.outside + 2 * d) = u32x4{v[c][0], v[c][1], v[c][2], v[c][3]};
        } else {
            for (int n = 0; n < PIECE / 8; ++n) {
                const uint32_t x = v[c][2 * n], y = v[c][2 * n + 1];
                *reinterpret_cast<u32x4*>(r.outside + 2 * d + 16 * n) =
                    u32x4{T::template from_fp8<false>(x, scale), T::template from_fp8<true>(x, scale),
                          T::template from_fp8<false>(y, scale), T::template from_fp8<true>(y, scale)};
            }
        }
    }
}

template <typename T, bool FP8>
__global__ __launch_bounds__(256) void cache_read_any_kernel(const Args a) {
    uint32_t group;
    const Side& s = side_of(a, group);
    const Row r = locate(a, s, group);
    if (!r.ok) return;
    uint16_t* out = reinterpret_cast<uint16_t*>(r.outside);
    if constexpr (!FP8) {
        for (uint32_t d = r.lane; d < s.dim; d += s.lanes) out[d] = reinterpret_cast<const uint16_t*>(r.inside)[d];
    } else {
        const float scale = *r.scale;
        for (uint32_t d = r.lane; d < s.dim; d += s.lanes) {
            const uint32_t v = reinterpret_cast<const uint8_t*>(r.inside)[d];
            out[d] = (uint16_t)T::template from_fp8<false>(v, scale);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------

int fill_side(Side& s, const hfk_cache_plane& p, const hfk_token_rows& r, uint64_t n, uint32_t piece) {
    if (p.head_dim > kMaxHeadDim) return HFK_ERR_TOO_LARGE;
    if (n * p.heads > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    const int64_t bytes = hfk::type_bytes(p.type);
    s.rows = static_cast<char*>(r.data);
    s.values = static_cast<char*>(p.values);
    s.scales = p.type == HFK_FP8_E4M3 ? p.scales : nullptr;
    s.row_token = 2 * r.token_stride;
    s.row_head = 2 * r.head_stride;
    s.block = bytes * p.block_stride;
    s.token = bytes * p.token_stride;
    s.head = bytes * p.head_stride;
    s.scale_block = p.scale_block_stride;
    s.scale_token = p.scale_token_stride;
    s.scale_head = p.scale_head_stride;
    s.heads = BlockSplit::of(p.heads);
    s.dim = p.head_dim;
    s.n_rows = (uint32_t)(n * p.heads);
    const uint32_t pieces = (p.head_dim + piece - 1u) / piece, most = piece == 16u ? 16u : 64u;
    s.lanes = 1;
    while (s.lanes < pieces && s.lanes < most) s.lanes *= 2u;
    return HFK_OK;
}

int check_side(const hfk_cache_plane& p, const hfk_token_rows& r, uint64_t n) {
    int rc = hfk::check_plane(p);
    if (rc == HFK_OK) rc = hfk::check_rows(r, n);
    if (rc != HFK_OK) return rc;
    return p.type == HFK_FP8_E4M3 || p.type == r.type ? HFK_OK : HFK_ERR_BAD_TYPE;
}

// Values per lane and step: 1 where rows have to be taken value by value.
uint32_t piece_of(const hfk_cache_plane& p, const hfk_token_rows& r) {
    if (!hfk::rows_aligned(r)) return 1;
    if (p.type == HFK_FP8_E4M3 && p.head_dim % 16u == 0 && hfk::plane_aligned(p, 16)) return 16;
    return p.head_dim % 8u == 0 && hfk::plane_aligned(p, p.type == HFK_FP8_E4M3 ? 8 : 16) ? 8 : 1;
}

// From this much read and written on, cache_read reads past the caches. Microseconds of a call, and of the call with a
// kernel behind it that reads the rows (keys and values of 8 heads of 128, e4m3 into bf16; through the caches | past them):
//   8192 tokens, 51 MB: 12.0, 42.8 | 14.5, 46.1;  16384, 102 MB: 25.5, 63.3 | 22.9, 62.5;  32768, 204 MB: 45.4, 106 | 42.4, 98.
// The same of bf16 caches, with a sum of the rows behind it:
//   8192 tokens, 67 MB: 12.0, 20.7 | 14.5, 23.2;  12288, 101 MB: 20.6, 32.7 | 19.5, 31.4;  32768, 268 MB: 52.0, 84.2 | 49.4, 81.3.
constexpr uint64_t kStreamBytes = 96ull << 20;

uint64_t moved_bytes(const Args& a, bool fp8) {
    return (uint64_t)a.side[0].n_rows * a.side[0].dim * (fp8 ? 3 : 4) + (uint64_t)a.side[1].n_rows * a.side[1].dim * (fp8 ? 3 : 4);
}

template <bool WRITE, typename T, bool FP8, int PIECE, int CHUNKS>
void launch_pieces(const Args& a, uint32_t grid, hipStream_t s) {
    if constexpr (WRITE) cache_write_kernel<T, FP8, PIECE, CHUNKS><<<grid, 256, 0, s>>>(a);
    else if (moved_bytes(a, FP8) < kStreamBytes) cache_read_kernel<T, FP8, PIECE, CHUNKS, false><<<grid, 256, 0, s>>>(a);
    else cache_read_kernel<T, FP8, PIECE, CHUNKS, true><<<grid, 256, 0, s>>>(a);
}

template <bool WRITE, typename T, bool FP8>
void launch_typed(const Args& a, uint32_t piece, uint32_t chunks, uint32_t grid, hipStream_t s) {
    if (piece == 1) {
        if constexpr (WRITE) cache_write_any_kernel<T, FP8><<<grid, 256, 0, s>>>(a);
        else cache_read_any_kernel<T, FP8><<<grid, 256, 0, s>>>(a);
        return;
    }
    if constexpr (FP8) {
        if (piece == 16) {      // lanes for 256 values: up to 1024 in four
            if (chunks == 1) launch_pieces<WRITE, T, FP8, 16, 1>(a, grid, s);
            else if (chunks == 2) launch_pieces<WRITE, T, FP8, 16, 2>(a, grid, s);
            else launch_pieces<WRITE, T, FP8, 16, 4>(a, grid, s);
            return;
        }
    }
    if (chunks == 1) launch_pieces<WRITE, T, FP8, 8, 1>(a, grid, s);
    else launch_pieces<WRITE, T, FP8, 8, 2>(a, grid, s);
}

template <bool WRITE>
int move_tokens(const hfk_cache_plane* kp, const hfk_token_rows* k, const hfk_cache_plane* vp, const hfk_token_rows* v,
                const int64_t* slots, uint64_t n, hfk_stream_t stream) {
    if (kp == nullptr || k == nullptr || (vp == nullptr) != (v == nullptr)) return HFK_ERR_NULL_POINTER;
    int rc = check_side(*kp, *k, n);
    if (rc != HFK_OK) return rc;
    if (vp != nullptr) {
        rc = check_side(*vp, *v, n);
        if (rc != HFK_OK) return rc;
        if (vp->type != kp->type || v->type != k->type) return HFK_ERR_BAD_TYPE;
        if (vp->blocks != kp->blocks || vp->block_tokens != kp->block_tokens) return HFK_ERR_BAD_SIZE;
    }
    if (n > 0x7fffffffull) return HFK_ERR_TOO_LARGE;
    if (n == 0 || kp->blocks == 0) return HFK_OK;
    if (slots == nullptr) return HFK_ERR_NULL_POINTER;
    uint32_t piece = piece_of(*kp, *k);
    if (vp != nullptr) {
        const uint32_t other = piece_of(*vp, *v);
        if (other < piece) piece = other;
    }
    Args a{};
    a.slots = slots;
    a.capacity = kp->blocks * kp->block_tokens;
    a.split = BlockSplit::of(kp->block_tokens);
    rc = fill_side(a.side[0], *kp, *k, n, piece);
    if (rc == HFK_OK && vp != nullptr) rc = fill_side(a.side[1], *vp, *v, n, piece);
    if (rc != HFK_OK) return rc;
    uint64_t groups[2] = {0, 0};
    uint32_t chunks = 1;
    for (int i = 0; i < (vp != nullptr ? 2 : 1); ++i) {
        const Side& s = a.side[i];
        const uint32_t per_group = 256u / s.lanes;
        groups[i] = ((uint64_t)s.n_rows + per_group - 1) / per_group;
        const uint32_t its = (s.dim + s.lanes * piece - 1u) / (s.lanes * piece);
        if (its > chunks) chunks = its;
    }
    if (!hfk::launch_fits(groups[0] + groups[1], 256)) return HFK_ERR_TOO_LARGE;
    a.first_groups = (uint32_t)groups[0];
    const uint32_t grid = (uint32_t)(groups[0] + groups[1]);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool fp8 = kp->type == HFK_FP8_E4M3;
    if (k->type == HFK_BF16) {
        if (fp8) launch_typed<WRITE, hfk::Bf16, true>(a, piece, chunks, grid, s);
        else launch_typed<WRITE, hfk::Bf16, false>(a, piece, chunks, grid, s);
    } else {
        if (fp8) launch_typed<WRITE, hfk::Fp16, true>(a, piece, chunks, grid, s);
        else launch_typed<WRITE, hfk::Fp16, false>(a, piece, chunks, grid, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? HFK_OK : (int)e;
}

}  // namespace

extern "C" {

int hfk_cache_write(const hfk_cache_plane* k_plane, const hfk_token_rows* k, const hfk_cache_plane* v_plane,
                    const hfk_token_rows* v, const int64_t* slots, uint64_t n, hfk_stream_t stream) {
    return move_tokens<true>(k_plane, k, v_plane, v, slots, n, stream);
}

int hfk_cache_read(const hfk_cache_plane* k_plane, const hfk_token_rows* k, const hfk_cache_plane* v_plane,
                   const hfk_token_rows* v, const int64_t* slots, uint64_t n, hfk_stream_t stream) {
    return move_tokens<false>(k_plane, k, v_plane, v, slots, n, stream);
}

}  // extern "C"
