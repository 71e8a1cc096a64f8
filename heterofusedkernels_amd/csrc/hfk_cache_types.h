// What the cache and attention kernels share: element types, conversions to and from them, the address of a token
// in a paged plane, and the host-side checks of a plane.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "hfk.h"

namespace hfk {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The two 16-bit types, as the kernels see them: bits in memory, floats in registers.
struct Bf16 {
    using Elem = __bf16;
    using Vec8 = bf16x8;
    static __device__ float to_float(uint32_t bits16) { return __uint_as_float(bits16 << 16); }
    static __device__ uint32_t pack2(float a, float b) {   // to nearest even
        bf16x2 p;
        p[0] = (__bf16)a;
        p[1] = (__bf16)b;
        return __builtin_bit_cast(uint32_t, p);
    }
    // Two e4m3 values of a dword's low or high half times a power of two: exact.
    template <bool HIGH>
    static __device__ uint32_t from_fp8(uint32_t four, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, HIGH));
    }
    static __device__ f32x4 mfma16(Vec8 a, Vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ f32x16 mfma32(Vec8 a, Vec8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static constexpr uint32_t kExponent = 0x7f80u;   // all ones in an infinity or a NaN
    static constexpr float kMostWeight = 0.0f;       // log2 of what a softmax weight may be lifted to: see below
};

struct Fp16 {
    using Elem = _Float16;
    using Vec8 = f16x8;
    static __device__ float to_float(uint32_t bits16) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16); }
    static __device__ uint32_t pack2(float a, float b) {
        f16x2 p;
        p[0] = (_Float16)a;
        p[1] = (_Float16)b;
        return __builtin_bit_cast(uint32_t, p);
    }
    // As above. From a scale of 2^8 on the product can pass fp16's range (e4m3 itself has no infinity): it becomes
    // the largest finite value, whose bits are one below infinity's.
    template <bool HIGH>
    static __device__ uint32_t from_fp8(uint32_t four, float scale) {
        uint32_t p = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, scale, HIGH));
        if (scale >= 256.0f) {
            if ((p & 0x7fffu) == 0x7c00u) p -= 1u;
            if ((p & 0x7fff0000u) == 0x7c000000u) p -= 0x10000u;
        }
        return p;
    }
    static __device__ f32x4 mfma16(Vec8 a, Vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ f32x16 mfma32(Vec8 a, Vec8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static constexpr uint32_t kExponent = 0x7c00u;
    // fp16 ends at 2^-24: weights are lifted so that the largest is 2^14, or thousands of small ones would vanish
    // from the second product though not from the sum.
    static constexpr float kMostWeight = 14.0f;
};

// index / T and index % T for block sizes that mostly are powers of two.
struct BlockSplit {
    uint32_t T;
    int32_t shift;   // log2(T), or -1
    __host__ __device__ static BlockSplit of(uint32_t T) {
        BlockSplit s{T, -1};
        for (int32_t b = 0; b < 32; ++b)
            if ((1u << b) == T) s.shift = b;
        return s;
    }
    __host__ __device__ uint64_t block(uint64_t slot) const { return shift >= 0 ? slot >> shift : slot / T; }
    __host__ __device__ uint32_t block32(uint32_t token) const { return shift >= 0 ? token >> shift : token / T; }
};

// ---- host-side checks ----------------------------------------------------------

inline bool known_type(uint32_t t) { return t == HFK_BF16 || t == HFK_FP16 || t == HFK_FP8_E4M3; }
inline uint32_t type_bytes(uint32_t t) { return t == HFK_FP8_E4M3 ? 1u : 2u; }
inline bool multiple_of(const void* p, uint64_t n) { return (uint64_t)(uintptr_t)p % n == 0; }

// Strides come from the caller and are only ever multiplied by indices inside the plane; bounding them keeps those
// products inside 64 bits.
inline bool stride_fits(int64_t s) { return s >= 0 && s < (1ll << 40); }

// A launch's threads are counted in 32 bits.
inline bool launch_fits(uint64_t groups, uint32_t threads) { return groups * threads < (1ull << 32); }

inline int check_plane(const hfk_cache_plane& p) {
    if (!known_type(p.type)) return HFK_ERR_BAD_TYPE;
    if (p.block_tokens == 0 || p.heads == 0 || p.head_dim == 0) return HFK_ERR_BAD_SIZE;
    if (p.heads > 65535u) return HFK_ERR_TOO_LARGE;
    if (p.blocks > (1ull << 31) || p.block_tokens > (1u << 30) || p.blocks * p.block_tokens > (1ull << 48)) return HFK_ERR_TOO_LARGE;
    if (!stride_fits(p.block_stride) || !stride_fits(p.token_stride) || !stride_fits(p.head_stride)) return HFK_ERR_BAD_SIZE;
    if (p.blocks != 0 && p.values == nullptr) return HFK_ERR_NULL_POINTER;
    if (p.type == HFK_FP8_E4M3) {
        if (p.blocks != 0 && p.scales == nullptr) return HFK_ERR_NULL_POINTER;
        if (!multiple_of(p.scales, 4)) return HFK_ERR_BAD_ALIGNMENT;
        if (!stride_fits(p.scale_block_stride) || !stride_fits(p.scale_token_stride) || !stride_fits(p.scale_head_stride))
            return HFK_ERR_BAD_SIZE;
    } else if (!multiple_of(p.values, 2)) {
        return HFK_ERR_BAD_ALIGNMENT;
    }
    return HFK_OK;
}

inline int check_rows(const hfk_token_rows& r, uint64_t n) {
    if (r.type != HFK_BF16 && r.type != HFK_FP16) return HFK_ERR_BAD_TYPE;
    if (n != 0 && r.data == nullptr) return HFK_ERR_NULL_POINTER;
    if (!multiple_of(r.data, 2)) return HFK_ERR_BAD_ALIGNMENT;
    if (!stride_fits(r.token_stride) || !stride_fits(r.head_stride)) return HFK_ERR_BAD_SIZE;
    return HFK_OK;
}

// All of a plane's (or of rows') addresses are multiples of `bytes` when its pointer and strides are.
inline bool plane_aligned(const hfk_cache_plane& p, uint64_t bytes) {
    const uint64_t e = bytes / type_bytes(p.type);
    return multiple_of(p.values, bytes) && (uint64_t)p.block_stride % e == 0 && (uint64_t)p.token_stride % e == 0 &&
           (uint64_t)p.head_stride % e == 0;
}

inline bool rows_aligned(const hfk_token_rows& r) {
    return multiple_of(r.data, 16) && (uint64_t)r.token_stride % 8 == 0 && (uint64_t)r.head_stride % 8 == 0;
}

}  // namespace hfk
