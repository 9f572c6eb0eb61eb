// A key / value cache in 4 bits: new tokens into it, entries read back, and entries dropped by the attention that they got.
#include "cache4.h"

namespace ti8 {
namespace cache4 {

namespace {

struct Rows {       // bf16 [batch][tokens][heads][dim], element strides, the last dim dense
    const uint16_t* p;
    int64_t sb, st, sh;
};

constexpr int TILE = 16;        // tokens per wave

// Eight elements per lane: the 32 that share a scale are four neighbouring lanes'.  a = max |x|; e = the exponent byte of the smallest
// 2^(e - 127) with a <= 6 * 2^(e - 127) = 1.5 * 2^(e - 125): that of a less two, one more where a's fraction is over 1.5.  Dividing by a power of two
// is exact, so codes do not depend on how the division is carried out.
__global__ __launch_bounds__(64) void append_kernel(const Cache c, const int32_t* starts, const int32_t* counts, int tokens, Rows k, Rows v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int lanes = c.dim >> 3, per = 64 / lanes;        // lanes of a row; rows of an instruction
    const int tiles = (tokens + TILE - 1) / TILE;
    const int t0 = (int)(blockIdx.x % tiles) * TILE, h = (int)(blockIdx.x / tiles) % c.heads, b = (int)(blockIdx.x / tiles) / c.heads;
    const int n = count_of(counts, b, tokens), start = start_of(starts, b);
    const int lane = threadIdx.x, chunk = lane % lanes;
    for (int t = t0 + lane / lanes; t < min(t0 + TILE, n); t += per) {
        const int page = page_of(c, b, start + t);
        if (page < 0) continue;
        uint8_t* const block = block_of(c, page, h);
        const int row = (start + t) & (c.page - 1);
#pragma unroll
        for (int values = 0; values < 2; ++values) {
            const Rows& x = values ? v : k;
            const uint4 w = *reinterpret_cast<const uint4*>(x.p + b * x.sb + t * x.st + h * x.sh + chunk * 8);
            float f[8] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y), bf16_lo(w.z), bf16_hi(w.z), bf16_lo(w.w), bf16_hi(w.w)};
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = f[i] == f[i] ? f[i] : 0.0f;
                amax = fmaxf(amax, fabsf(f[i]));
            }
            amax = dpp_max<0x4E>(dpp_max<0xB1>(amax));
            const int e = min(max((int)((__float_as_uint(amax) + 0x3fffffu) >> 23) - 2, 1), 252);
            *reinterpret_cast<uint32_t*>(block + idx::cache4_codes(c.page, c.dim, values, row) + chunk * 4) = encode8(f, scale_of(e));
            if ((chunk & 3) == 0) block[idx::cache4_scales(c.page, c.dim, values, row) + (chunk >> 2)] = (uint8_t)e;
        }
        if (c.weights && chunk == 0) c.weights[((int64_t)page * c.heads + h) * c.page + row] = 0.0f;
    }
#endif
}

__global__ __launch_bounds__(64) void read_kernel(const Cache c, const int32_t* starts, const int32_t* counts, int tokens, uint16_t* k, uint16_t* v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int lanes = c.dim >> 3, per = 64 / lanes;
    const int tiles = (tokens + TILE - 1) / TILE;
    const int t0 = (int)(blockIdx.x % tiles) * TILE, h = (int)(blockIdx.x / tiles) % c.heads, b = (int)(blockIdx.x / tiles) / c.heads;
    const int n = count_of(counts, b, tokens), start = start_of(starts, b);
    const int lane = threadIdx.x, chunk = lane % lanes;
    for (int t = t0 + lane / lanes; t < min(t0 + TILE, tokens); t += per) {
        const int page = t < n ? page_of(c, b, start + t) : -1, row = (start + t) & (c.page - 1);
        const uint8_t* const block = block_of(c, max(page, 0), h);
#pragma unroll
        for (int values = 0; values < 2; ++values) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (page >= 0)
                x = decode8(*reinterpret_cast<const uint32_t*>(block + idx::cache4_codes(c.page, c.dim, values, row) + chunk * 4),
                            scale_of(block[idx::cache4_scales(c.page, c.dim, values, row) + (chunk >> 2)]));
            *reinterpret_cast<uint4*>((values ? v : k) + (((int64_t)b * tokens + t) * c.heads + h) * c.dim + chunk * 8) = x;
        }
    }
#endif
}

// order of the weights as unsigned numbers: -0 is 0, NaN the largest
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SELECT = 1024;        // threads

// Which entries of a (sequence, head) stay: one workgroup each.  The `heavy`-th largest weight of the old entries is found byte by byte from the
// top (a histogram of those that agree so far), then the entries are gone through in order: those above it stay, and the first of those equal to it.
__global__ __launch_bounds__(SELECT) void select_kernel(const Cache c, const int32_t* lengths, int keep, int recent, int32_t* kept, int32_t* new_lengths) {
    __shared__ int bins[256], found[2], sums[2][SELECT / 64];
    const int b = blockIdx.x / c.heads, h = blockIdx.x % c.heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = length_of(c, lengths, b), stay = min(n, keep);
    int32_t* const mine = kept + ((int64_t)b * c.heads + h) * keep;
    if (h == 0 && tid == 0) new_lengths[b] = stay;
    for (int i = stay + tid; i < keep; i += SELECT) mine[i] = -1;
    if (n <= keep) {
        for (int i = tid; i < n; i += SELECT) mine[i] = i;
        return;
    }
    const int old = n - min(recent, n), heavy = stay - (n - old);
    const auto order = [&](int j) {
        const int page = page_of(c, b, j);
        return page < 0 ? 0u : order_of(c.weights[((int64_t)page * c.heads + h) * c.page + (j & (c.page - 1))]);
    };
    uint32_t limit = 0;         // the heavy-th largest, as far as it is known
    int left = heavy;           // how many of those that agree with it so far are to stay
    if (heavy > 0)
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
            for (int j = tid; j < old; j += SELECT) {
                const uint32_t u = order(j);
                if (shift == 24 || u >> (shift + 8) == limit >> (shift + 8)) atomicAdd(&bins[u >> shift & 255], 1);
            }
            __syncthreads();
            if (wave == 0) {        // lane l has bins 255 - 4 l .. 252 - 4 l, from the largest on
                int own[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += own[i] = bins[255 - 4 * lane - i];
                int before = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int x = __shfl_up(before, d, 64);
                    if (lane >= d) before += x;
                }
                before -= sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < left && before + own[i] >= left) {
                        found[0] = 255 - 4 * lane - i;
                        found[1] = left - before;
                    }
                    before += own[i];
                }
            }
            __syncthreads();
            limit |= (uint32_t)found[0] << shift;
            left = found[1];
        }
    int out = 0, equals = 0;        // entries that stay, and entries equal to the limit, so far
    for (int j0 = 0; j0 < old && heavy > 0; j0 += SELECT) {
        const uint32_t u = j0 + tid < old ? order(j0 + tid) : 0u;
        const bool equal = j0 + tid < old && u == limit, above = j0 + tid < old && u > limit;
        const uint64_t e = __ballot(equal), a = __ballot(above), below = (1ull << lane) - 1;
        if (lane == 0) {
            sums[0][wave] = __popcll(e);
            sums[1][wave] = __popcll(a);
        }
        __syncthreads();
        int eq = equals + __popcll(e & below), ab = __popcll(a & below);
        for (int w = 0; w < SELECT / 64; ++w) {
            if (w < wave) {
                eq += sums[0][w];
                ab += sums[1][w];
            }
        }
        // of the equal ones in front min(eq, left) stay
        const int place = out + ab + min(eq, left) - min(equals, left);
        if (above || (equal && eq < left)) mine[place] = j0 + tid;
        int total_e = 0, total_a = 0;
        for (int w = 0; w < SELECT / 64; ++w) {
            total_e += sums[0][w];
            total_a += sums[1][w];
        }
        out += total_a + min(equals + total_e, left) - min(equals, left);
        equals += total_e;
        __syncthreads();
    }
    for (int j = old + tid; j < n; j += SELECT) mine[heavy + j - old] = j;
}

constexpr int MOVE = 64;        // entries per workgroup

__global__ __launch_bounds__(256) void move_kernel(const Cache c, const int32_t* kept, const int32_t* new_table, int new_pages, int64_t new_stride, int keep) {
    const int blocks = (keep + MOVE - 1) / MOVE;
    const int i0 = (int)(blockIdx.x % blocks) * MOVE, h = (int)(blockIdx.x / blocks) % c.heads, b = (int)(blockIdx.x / blocks) / c.heads;
    const int32_t* const mine = kept + ((int64_t)b * c.heads + h) * keep;
    const int words = c.dim / 8, pieces = words / 2 + 2;        // an entry: its codes 16 bytes at a time, keys and values, their scales; the weight
    for (int x = threadIdx.x; x < MOVE * pieces; x += 256) {
        const int i = i0 + x / pieces, piece = x % pieces;
        if (i >= keep) break;
        const int j = mine[i];
        if (j < 0) break;
        const int from = page_of(c, b, j), to = (i >> c.log2_page) < new_pages ? new_table[b * new_stride + (i >> c.log2_page)] : -1;
        if (from < 0 || (unsigned)to >= (unsigned)c.pages) continue;
        const uint8_t* const src = block_of(c, from, h);
        uint8_t* const dst = block_of(c, to, h);
        const int r = j & (c.page - 1), s = i & (c.page - 1);
        if (piece < words / 2) {
            const int values = piece >= words / 4, at = (piece % (words / 4)) * 16;
            *reinterpret_cast<uint4*>(dst + idx::cache4_codes(c.page, c.dim, values, s) + at) =
                *reinterpret_cast<const uint4*>(src + idx::cache4_codes(c.page, c.dim, values, r) + at);
        } else {
            const int values = piece - words / 2;
            const int from_at = idx::cache4_scales(c.page, c.dim, values, r), to_at = idx::cache4_scales(c.page, c.dim, values, s);
            if (c.dim == 128) *reinterpret_cast<uint32_t*>(dst + to_at) = *reinterpret_cast<const uint32_t*>(src + from_at);
            else *reinterpret_cast<uint16_t*>(dst + to_at) = *reinterpret_cast<const uint16_t*>(src + from_at);
            if (!values) c.weights[((int64_t)to * c.heads + h) * c.page + s] = c.weights[((int64_t)from * c.heads + h) * c.page + r];
        }
    }
}

int check_rows(const char* fn, const char* name, const void* p, int64_t sb, int64_t st, int64_t sh) {
    if (!p) return fail(TI8_ERR_NULL, "%s: %s is required", fn, name);
    if (!aligned16(p) || sb % 8 || st % 8 || sh % 8) return fail(TI8_ERR_ALIGN, "%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", fn, name);
    return TI8_OK;
}

int check_tokens(const char* fn, const Cache& c, const int32_t* starts, int64_t tokens, int64_t tile, unsigned* grid) {
    if (!starts) return fail(TI8_ERR_NULL, "%s: starts is required", fn);
    if (tokens <= 0 || tokens > (1 << 30)) return fail(TI8_ERR_SHAPE, "%s: need 0 < tokens <= 2^30, got %lld", fn, (long long)tokens);
    const int64_t n = (int64_t)c.batch * c.heads * ((tokens + tile - 1) / tile);
    if (n > 0x7fffffff) return fail(TI8_ERR_SHAPE, "%s: %lld workgroups are more than a launch takes", fn, (long long)n);
    *grid = (unsigned)n;
    return TI8_OK;
}

}  // namespace

}  // namespace cache4
}  // namespace ti8

using namespace ti8;
using namespace ti8::cache4;

extern "C" int ti8_cache4_append(const ti8_cache4* p, const int32_t* starts, const int32_t* counts, int64_t tokens,
                                 const void* k, int64_t k_stride_b, int64_t k_stride_t, int64_t k_stride_h,
                                 const void* v, int64_t v_stride_b, int64_t v_stride_t, int64_t v_stride_h, ti8_stream_t stream) {
    const char* fn = "ti8_cache4_append";
    Cache c;
    unsigned grid;
    if (int e = check(fn, p, c)) return e;
    if (int e = check_tokens(fn, c, starts, tokens, TILE, &grid)) return e;
    if (int e = check_rows(fn, "k", k, k_stride_b, k_stride_t, k_stride_h)) return e;
    if (int e = check_rows(fn, "v", v, v_stride_b, v_stride_t, v_stride_h)) return e;
    const Rows rk{static_cast<const uint16_t*>(k), k_stride_b, k_stride_t, k_stride_h}, rv{static_cast<const uint16_t*>(v), v_stride_b, v_stride_t, v_stride_h};
    hipLaunchKernelGGL(append_kernel, dim3(grid), dim3(64), 0, static_cast<hipStream_t>(stream), c, starts, counts, (int)tokens, rk, rv);
    return check_launch(fn);
}

extern "C" int ti8_cache4_read(const ti8_cache4* p, const int32_t* starts, const int32_t* counts, int64_t tokens, void* k, void* v, ti8_stream_t stream) {
    const char* fn = "ti8_cache4_read";
    Cache c;
    unsigned grid;
    if (int e = check(fn, p, c)) return e;
    if (int e = check_tokens(fn, c, starts, tokens, TILE, &grid)) return e;
    if (int e = check_rows(fn, "k", k, 0, 0, 0)) return e;
    if (int e = check_rows(fn, "v", v, 0, 0, 0)) return e;
    hipLaunchKernelGGL(read_kernel, dim3(grid), dim3(64), 0, static_cast<hipStream_t>(stream), c, starts, counts, (int)tokens,
                       static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
    return check_launch(fn);
}

extern "C" int ti8_cache4_evict(const ti8_cache4* p, const int32_t* lengths, const int32_t* new_table, int64_t new_pages, int64_t new_stride,
                                int64_t keep, int64_t recent, int32_t* kept, int32_t* new_lengths, ti8_stream_t stream) {
    const char* fn = "ti8_cache4_evict";
    Cache c;
    if (int e = check(fn, p, c)) return e;
    if (!c.weights || !lengths || !new_table || !kept || !new_lengths) return fail(TI8_ERR_NULL, "%s: weights, lengths, new_table, kept and new_lengths are required", fn);
    if (keep <= 0 || keep > (1 << 30) || recent < 0 || recent > keep || new_pages <= 0 || new_pages > (1 << 30) / c.page || new_pages * c.page < keep || new_stride < new_pages)
        return fail(TI8_ERR_SHAPE, "%s: need 0 <= recent <= keep, 0 < keep <= new_pages * page_size <= 2^30 and new_stride >= new_pages; got keep=%lld recent=%lld "
                    "new_pages=%lld new_stride=%lld", fn, (long long)keep, (long long)recent, (long long)new_pages, (long long)new_stride);
    const int64_t moves = (int64_t)c.batch * c.heads * ((keep + MOVE - 1) / MOVE);
    if (moves > 0x7fffffff) return fail(TI8_ERR_SHAPE, "%s: %lld workgroups are more than a launch takes", fn, (long long)moves);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)(c.batch * c.heads)), dim3(SELECT), 0, st, c, lengths, (int)keep, (int)recent, kept, new_lengths);
    if (int e = check_launch(fn)) return e;
    hipLaunchKernelGGL(move_kernel, dim3((unsigned)moves), dim3(256), 0, st, c, kept, new_table, (int)new_pages, new_stride, (int)keep);
    return check_launch(fn);
}
