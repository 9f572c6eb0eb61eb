// Attention over a cache in 4 bits.
#include "cache4.h"

namespace ti8 {
namespace cache4 {

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int KEYS = 128;       // keys at a time, and threads of a workgroup

struct Args {
    Cache c;
    const int32_t *lengths, *counts;
    const uint16_t* q;
    int64_t q_sb, q_st, q_sh;
    uint16_t* out;
    float* lse;
    int tokens, heads, group;       // group = query heads per kv head
    float scale;
};

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ float dot(const uint8_t* block, const Cache& c, int row, const float* q) {
    float s = 0.0f;
    for (int w = 0; w < c.dim / 8; ++w) {
        const uint4 x = decode8(*reinterpret_cast<const uint32_t*>(block + idx::cache4_codes(c.page, c.dim, 0, row) + w * 4),
                                scale_of(block[idx::cache4_scales(c.page, c.dim, 0, row) + w / 4]));
        const float* p = q + w * 8;
        s = fmaf(bf16_lo(x.x), p[0], s); s = fmaf(bf16_hi(x.x), p[1], s); s = fmaf(bf16_lo(x.y), p[2], s); s = fmaf(bf16_hi(x.y), p[3], s);
        s = fmaf(bf16_lo(x.z), p[4], s); s = fmaf(bf16_hi(x.z), p[5], s); s = fmaf(bf16_lo(x.w), p[6], s); s = fmaf(bf16_hi(x.w), p[7], s);
    }
    return s;
}
#endif

// one row of queries per workgroup
__global__ __launch_bounds__(KEYS) void row_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float q[128], p[KEYS], part[2];
    const Cache& c = a.c;
    const int head = blockIdx.x % a.heads, t = (int)(blockIdx.x / a.heads) % a.tokens, b = (int)(blockIdx.x / a.heads) / a.tokens;
    const int h = head / a.group, tid = threadIdx.x, count = count_of(a.counts, b, a.tokens), length = length_of(c, a.lengths, b);
    const int sees = t < count ? max(length - count + t + 1, 0) : 0;
    if (tid < c.dim) q[tid] = bf16_lo(a.q[b * a.q_sb + t * a.q_st + head * a.q_sh + tid]);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const auto all = [&](float x, bool largest) {
        for (int d = 32; d; d >>= 1) { const float y = __shfl_xor(x, d, 64); x = largest ? fmaxf(x, y) : x + y; }
        __syncthreads();
        if ((tid & 63) == 0) part[tid >> 6] = x;
        __syncthreads();
        return largest ? fmaxf(part[0], part[1]) : part[0] + part[1];
    };
    for (int j0 = 0; j0 < sees; j0 += KEYS) {
        __syncthreads();
        const int j = j0 + tid, page = j < sees ? page_of(c, b, j) : -1;
        float s = -INFINITY;
        if (page >= 0) s = dot(block_of(c, page, h), c, j & (c.page - 1), q) * (a.scale * LOG2E);
        const float top = fmaxf(m, all(s, true)), from = top == -INFINITY ? 0.0f : top;
        const float e = exp2f(s - from);
        p[tid] = e;
        const float shrink = exp2f(m - from);
        l = l * shrink + all(e, false);
        m = top;
        if (tid < c.dim) {
            o *= shrink;
            for (int i = 0; i < min(KEYS, sees - j0); ++i) {
                const int page_i = page_of(c, b, j0 + i);
                if (page_i < 0) continue;
                const uint8_t* block = block_of(c, page_i, h);
                const int row = (j0 + i) & (c.page - 1);
                const uint32_t code = block[idx::cache4_codes(c.page, c.dim, 1, row) + tid / 2];
                const uint32_t x = decode<0>(code, scale_of(block[idx::cache4_scales(c.page, c.dim, 1, row) + tid / GROUP]));
                o = fmaf(p[i], tid & 1 ? bf16_hi(x) : bf16_lo(x), o);
            }
        }
    }
    const int64_t row = ((int64_t)b * a.tokens + t) * a.heads + head;
    if (tid < c.dim) a.out[row * c.dim + tid] = (uint16_t)f32_to_bf16_bits(l > 0.0f ? o / l : l);
    if (tid == 0) a.lse[row] = l > 0.0f ? (m + log2f(l)) * LN2 : l == 0.0f ? -INFINITY : l;
#endif
}

// one key per thread
__global__ __launch_bounds__(KEYS) void weights_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float q[128];
    const Cache& c = a.c;
    const int blocks = (c.capacity() + KEYS - 1) / KEYS;
    const int j = (int)(blockIdx.x % blocks) * KEYS + threadIdx.x, h = (int)(blockIdx.x / blocks) % c.heads, b = (int)(blockIdx.x / blocks) / c.heads;
    const int count = count_of(a.counts, b, a.tokens), length = length_of(c, a.lengths, b), page = j < length ? page_of(c, b, j) : -1;
    float sum = 0.0f;
    for (int t = 0; t < count; ++t)
        for (int g = 0; g < a.group; ++g) {
            const int head = h * a.group + g;
            __syncthreads();
            if (threadIdx.x < c.dim) q[threadIdx.x] = bf16_lo(a.q[b * a.q_sb + t * a.q_st + head * a.q_sh + threadIdx.x]);
            __syncthreads();
            if (page < 0 || j > length - count + t) continue;
            const float lse = a.lse[((int64_t)b * a.tokens + t) * a.heads + head] * LOG2E;
            sum += exp2f(dot(block_of(c, page, h), c, j & (c.page - 1), q) * (a.scale * LOG2E) - lse);
        }
    if (page >= 0) c.weights[((int64_t)page * c.heads + h) * c.page + (j & (c.page - 1))] += sum;
#endif
}

}  // namespace

}  // namespace cache4
}  // namespace ti8

using namespace ti8;
using namespace ti8::cache4;

extern "C" int64_t ti8_cache4_attention_workspace(const ti8_cache4* p, int64_t tokens, int64_t heads) {
    Cache c;
    if (check("ti8_cache4_attention_workspace", p, c)) return -1;
    if (tokens <= 0 || tokens > (1 << 24) || heads <= 0 || heads % c.heads || heads / c.heads > 4096 || c.batch * tokens * heads > 0x7fffffff ||
        (int64_t)c.batch * c.heads * ((c.capacity() + 127) / 128) > 0x7fffffff)
        return -1;
    return 0;
}

extern "C" int ti8_cache4_attention(const ti8_cache4* p, const int32_t* lengths, const int32_t* counts, int64_t tokens, int64_t heads,
                                    const void* q, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h, float scale, int accumulate,
                                    void* out, float* lse, void* workspace, int64_t workspace_bytes, ti8_stream_t stream) {
    const char* fn = "ti8_cache4_attention";
    Cache c;
    if (int e = check(fn, p, c)) return e;
    const int64_t need = ti8_cache4_attention_workspace(p, tokens, heads);
    if (need < 0) return fail(TI8_ERR_SHAPE, "%s: need tokens > 0 and heads a multiple of kv_heads, and no more rows than a launch takes; got tokens=%lld heads=%lld", fn,
                              (long long)tokens, (long long)heads);
    if (!q || !lengths || !out || !lse || (accumulate && !c.weights) || (need && !workspace))
        return fail(TI8_ERR_NULL, "%s: q, lengths, out and lse are required, the weights to add up as well, and the workspace", fn);
    if (need > workspace_bytes) return fail(TI8_ERR_SHAPE, "%s: %lld bytes of workspace are needed, got %lld", fn, (long long)need, (long long)workspace_bytes);
    if (!aligned16(q) || !aligned16(out) || (reinterpret_cast<uintptr_t>(lse) & 3) || !aligned16(workspace) || q_stride_b % 8 || q_stride_t % 8 || q_stride_h % 8)
        return fail(TI8_ERR_ALIGN, "%s: q, out and the workspace must be 16-byte aligned, q's strides multiples of 8 elements", fn);
    const Args a{c, lengths, counts, static_cast<const uint16_t*>(q), q_stride_b, q_stride_t, q_stride_h, static_cast<uint16_t*>(out), lse,
                 (int)tokens, (int)heads, (int)(heads / c.heads), scale};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(row_kernel, dim3((unsigned)(c.batch * tokens * heads)), dim3(KEYS), 0, st, a);
    if (int e = check_launch(fn)) return e;
    if (accumulate) hipLaunchKernelGGL(weights_kernel, dim3((unsigned)((int64_t)c.batch * c.heads * ((c.capacity() + KEYS - 1) / KEYS))), dim3(KEYS), 0, st, a);
    return check_launch(fn);
}
