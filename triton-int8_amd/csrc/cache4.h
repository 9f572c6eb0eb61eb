// What the kernels of the 4-bit cache share: its description on the device, 4-bit floats, the checks of an entry point.
#pragma once
#include "ti8_common.h"
#include "index_math.h"

namespace ti8 {
namespace cache4 {

constexpr int GROUP = 32;       // elements that share a scale

struct Cache {
    uint8_t* pool;
    const int32_t* table;
    float* weights;
    int64_t table_stride;
    int pages, heads, page, log2_page, dim, block_bytes, batch, table_pages;
    __host__ __device__ __forceinline__ int capacity() const { return table_pages << log2_page; }
};

inline bool page_size_ok(int64_t n) { return n >= 16 && n <= 256 && (n & (n - 1)) == 0; }

// null pointers are the entry points' own business where a part is optional
inline int check(const char* fn, const ti8_cache4* c, Cache& out) {
    if (!c || !c->pool || !c->table) return fail(TI8_ERR_NULL, "%s: cache, pool and table are required", fn);
    if ((c->head_dim != 64 && c->head_dim != 128) || !page_size_ok(c->page_size))
        return fail(TI8_ERR_SHAPE, "%s: need head_dim 64 or 128 and page_size 16, 32, 64, 128 or 256; got head_dim=%lld page_size=%lld", fn,
                    (long long)c->head_dim, (long long)c->page_size);
    // entries are counted in 31 bits
    if (c->batch <= 0 || c->batch > 65535 || c->kv_heads <= 0 || c->kv_heads > 65535 || c->pages <= 0 || c->pages > 0x7fffffff || c->table_pages <= 0 ||
        c->table_pages > (1 << 30) / c->page_size || c->table_stride < c->table_pages)
        return fail(TI8_ERR_SHAPE, "%s: need batch, kv_heads in 1 .. 65535, pages > 0, 0 < table_pages * page_size <= 2^30 and table_stride >= table_pages; "
                    "got batch=%lld kv_heads=%lld pages=%lld table_pages=%lld table_stride=%lld", fn, (long long)c->batch, (long long)c->kv_heads,
                    (long long)c->pages, (long long)c->table_pages, (long long)c->table_stride);
    if (!aligned16(c->pool) || (reinterpret_cast<uintptr_t>(c->table) & 3) || (reinterpret_cast<uintptr_t>(c->weights) & 3))
        return fail(TI8_ERR_ALIGN, "%s: the pool must be 16-byte aligned, table and weights 4-byte", fn);
    out.pool = static_cast<uint8_t*>(c->pool);
    out.table = c->table;
    out.weights = c->weights;
    out.table_stride = c->table_stride;
    out.pages = (int)c->pages;
    out.heads = (int)c->kv_heads;
    out.page = (int)c->page_size;
    out.log2_page = idx::log2_of((int)c->page_size);
    out.dim = (int)c->head_dim;
    out.block_bytes = idx::cache4_block_bytes((int)c->page_size, (int)c->head_dim);
    out.batch = (int)c->batch;
    out.table_pages = (int)c->table_pages;
    return TI8_OK;
}

// page of entry j of sequence b, or -1 where there is none
__device__ __forceinline__ int page_of(const Cache& c, int b, int j) {
    if (j < 0 || j >= c.capacity()) return -1;
    const int p = c.table[b * c.table_stride + (j >> c.log2_page)];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}
__device__ __forceinline__ uint8_t* block_of(const Cache& c, int page, int head) { return c.pool + ((int64_t)page * c.heads + head) * c.block_bytes; }

// length and number of new tokens of a sequence, as far as the table has room
__device__ __forceinline__ int length_of(const Cache& c, const int32_t* lengths, int b) { return min(max(lengths[b], 0), c.capacity()); }
// (cut so that a token's number added to it stays in 32 bits)
__device__ __forceinline__ int start_of(const int32_t* starts, int b) { return min(max(starts[b], -(1 << 30)), 1 << 30); }
__device__ __forceinline__ int count_of(const int32_t* counts, int b, int tokens) { return counts ? min(max(counts[b], 0), tokens) : tokens; }

// v plus the number of the lane that DPP control CTRL names, in the rows of ROW_MASK, where there is such a lane
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false); }
// sums over the lanes up to this one: row_shr 1, 2, 4 and 8 within rows of 16, then row_bcast:15 and row_bcast:31 (no LDS traffic: six shuffles
// take 0.3 us of a kernel's beginning)
__device__ __forceinline__ int wave_prefix(int v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}

// 16 bytes that nobody asks for again soon
__device__ __forceinline__ uint4 stream_load(const void* p) { return __builtin_bit_cast(uint4, __builtin_nontemporal_load(static_cast<const v4i*>(p))); }
__device__ __forceinline__ void stream_store(void* p, uint4 x) { __builtin_nontemporal_store(__builtin_bit_cast(v4i, x), static_cast<v4i*>(p)); }

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
#if defined(__HIP_DEVICE_COMPILE__)
// the two bf16 that byte I of a word of codes stands for (v_cvt_scalef32_pk_bf16_fp4)
template <int I>
__device__ __forceinline__ uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}
__device__ __forceinline__ uint4 decode8(uint32_t codes, float scale) {
    return make_uint4(decode<0>(codes, scale), decode<1>(codes, scale), decode<2>(codes, scale), decode<3>(codes, scale));
}
// eight values as codes of value / scale, to the nearest, of two the even one (v_cvt_scalef32_pk_fp4_f32)
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], float scale) {
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}
#endif

}  // namespace cache4
}  // namespace ti8
