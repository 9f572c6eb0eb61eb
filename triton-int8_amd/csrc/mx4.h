// 4-bit floats with shared scales ("mx4"): what the quantisers, the norm and the product of that format share.
//
// 32 neighbouring elements x of a row share the scale 2^(e - 127), e the smallest of 1 .. 252 with max |x| <= 6 * 2^(e - 127) (252 where there is none, so that
// every value is finite in bf16: what is beyond 1.5 * 2^127 counts as that); an element's code is the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} to x / scale, of
// two that are as near the one with the even code.  e = 255 (and codes of zero): the group holds an infinity or a NaN, and stands for NaN, which a product
// hands on.
#pragma once
#include "ti8_common.h"
#include "index_math.h"

namespace ti8 {
namespace mx4 {

constexpr uint32_t NAN_SCALE = 255;

struct Tensor {
    uint8_t *codes, *scales;
    int64_t ld, scale_ld;
};

inline int check(const char* fn, const char* name, const ti8_mx4* t, int64_t rows, int64_t cols, Tensor& out) {
    if (!t->codes || !t->scales) return fail(TI8_ERR_NULL, "%s: codes and scales of %s are required", fn, name);
    const int64_t tiles = idx::mx4_tiles(cols);
    if (t->ld < tiles * idx::MX4_TILE_BYTES || t->scale_ld < rows * idx::MX4_TILE_SCALES)
        return fail(TI8_ERR_SHAPE, "%s: %lld x %lld elements of %s need ld >= %lld and scale_ld >= %lld, got %lld and %lld", fn, (long long)rows, (long long)cols, name,
                    (long long)(tiles * idx::MX4_TILE_BYTES), (long long)(rows * idx::MX4_TILE_SCALES), (long long)t->ld, (long long)t->scale_ld);
    if (!aligned16(t->codes) || t->ld % 16 || (reinterpret_cast<uintptr_t>(t->scales) & 7) || t->scale_ld % 8)
        return fail(TI8_ERR_ALIGN, "%s: codes of %s must be 16-byte aligned and its scales 8-byte, ld and scale_ld multiples of that", fn, name);
    out = Tensor{static_cast<uint8_t*>(t->codes), static_cast<uint8_t*>(t->scales), t->ld, t->scale_ld};
    return TI8_OK;
}

#if defined(__HIP_DEVICE_COMPILE__)
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// 16 bytes at any even address: rows of bf16 tensors start wherever their strides put them
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wcast-align"
__device__ __forceinline__ uint4 load16(const uint16_t* p) { return __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4_any*>(p)); }
__device__ __forceinline__ void store16(uint16_t* p, const uint4& v) { *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, v); }
// The same past the caches, for what nobody reads again soon and what a kernel reads once; what is in the caches is found there.  Quantised both ways, through them /
// past them, tensors from memory: 4096 x 4096 16.2 us / 13.3, 14336 x 4096 42 / 37; just written by another kernel 12.0 / 11.5, 16384 x 4096 44 / 31
__device__ __forceinline__ uint4 load16_once(const uint16_t* p) { return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p))); }
__device__ __forceinline__ void stream16(uint16_t* p, const uint4& v) { __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4_any*>(p)); }
#pragma clang diagnostic pop
// Elements col .. col + 7 of a row of `cols` elements (at least 8), zeros for those that it does not have; without a branch, so that several are on their way at
// once: what lies across the row's end is read from its last eight and shifted.
__device__ __forceinline__ uint4 load8_of(const uint16_t* row, int64_t col, int64_t cols) {
    const int64_t left = cols - col;
    uint4 v = load16_once(row + (left >= 8 ? col : left > 0 ? cols - 8 : 0));
    const int gone = left >= 8 ? 0 : left > 0 ? 8 - (int)left : 8;
    if (gone & 4) v = make_uint4(v.z, v.w, 0, 0);
    if (gone & 2) v = make_uint4(v.y, v.z, v.w, 0);
    if (gone & 1) v = make_uint4((v.x >> 16) | (v.y << 16), (v.y >> 16) | (v.z << 16), (v.z >> 16) | (v.w << 16), v.w >> 16);
    if (gone == 8) v = make_uint4(0, 0, 0, 0);
    return v;
}
// the same of rows of up to 7 elements
__device__ __forceinline__ uint4 load_short(const uint16_t* row, int64_t col, int64_t cols) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (col + j < cols) w[j >> 1] |= (uint32_t)row[col + j] << (16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// N rows from `row0` on, `step` apart, zeros where there are none.  `split`: the lanes' octets may lie across the rows' end.
template <int N>
__device__ __forceinline__ void load_rows(uint4 (&v)[N], const uint16_t* x, int64_t ldx, int64_t row0, int step, int64_t rows, int64_t col, int64_t cols, bool split) {
    if (!split) {
        const int64_t at = col < cols ? col : cols - 8;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t row = row0 + i * step;
            v[i] = load16_once(x + (row < rows ? row : rows - 1) * ldx + at);
        }
    } else if (cols >= 8) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t row = row0 + i * step;
            v[i] = load8_of(x + (row < rows ? row : rows - 1) * ldx, col, cols);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t row = row0 + i * step;
            v[i] = load_short(x + (row < rows ? row : rows - 1) * ldx, col, cols);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (row0 + i * step >= rows || col >= cols) v[i] = make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v, int64_t left) {
    if (left >= 8) return store16(p, v);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) p[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
}

// Magnitudes of bf16 as integers: ordered as the numbers, infinities and NaN above them all
constexpr uint32_t MAGNITUDE = 0x7fff7fffu;
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t largest2(const uint4& v) {
    return pk_max(pk_max(v.x & MAGNITUDE, v.y & MAGNITUDE), pk_max(v.z & MAGNITUDE, v.w & MAGNITUDE));
}
__device__ __forceinline__ uint32_t halves_max(uint32_t m) { return max(m & 0xffffu, m >> 16); }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) { return max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false)); }
// pk_max over the lanes whose numbers differ in bit 4 or bit 5, in all of them
__device__ __forceinline__ uint32_t pk_max_16(uint32_t m) {
    const auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    return pk_max(r[0], r[1]);
}
__device__ __forceinline__ uint32_t pk_max_32(uint32_t m) {
    const auto r = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return pk_max(r[0], r[1]);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_pk_max(uint32_t v) { return pk_max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false)); }
// over four neighbouring lanes, in all of them
__device__ __forceinline__ uint32_t quad_max(uint32_t v) { return dpp_umax<0x4E>(dpp_umax<0xB1>(v)); }

// the scale byte of a group whose largest magnitude is the bf16 `m`: its exponent less 2, one more where its fraction is over 1.5
__device__ __forceinline__ uint32_t scale_byte(uint32_t m) {
    const int e = (int)(((m << 16) + 0x3fffffu) >> 23) - 2;
    return m >= 0x7f80u ? NAN_SCALE : (uint32_t)min(max(e, 1), 252);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

template <int I>
__device__ __forceinline__ uint32_t encode2(uint32_t old, uint32_t pair, float scale) {     // (v_cvt_scalef32_pk_fp4_bf16: to the nearest, of two the even one)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(ti8_bf16x2, pair), scale, I);
}
// eight neighbouring elements as codes, the first in the low bits
__device__ __forceinline__ uint32_t encode8(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t byte) {
    const float scale = scale_of(byte);
    const uint32_t w = encode2<3>(encode2<2>(encode2<1>(encode2<0>(0u, a, scale), b, scale), c, scale), d, scale);
    return byte == NAN_SCALE ? 0u : w;
}
// four of them
__device__ __forceinline__ uint32_t encode4(uint32_t a, uint32_t b, uint32_t byte) {
    const float scale = scale_of(byte);
    const uint32_t w = encode2<1>(encode2<0>(0u, a, scale), b, scale);
    return byte == NAN_SCALE ? 0u : w;
}
#endif

}  // namespace mx4
}  // namespace ti8
