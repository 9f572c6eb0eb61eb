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
// Bound by memory: a wave has the keys and values of all its 16 tokens in flight before it converts the first, and past the caches, which they would only
// fill (4 x 4096 tokens of 32 heads 67 us, 5.0 TB/s; through the caches 90; read back 50 us, 6.8 TB/s, and 82).
template <int D>
__global__ __launch_bounds__(64) void append_kernel(const Cache c, const int32_t* starts, const int32_t* counts, int tokens, Rows k, Rows v) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 8, PER = 64 / LANES, ROUNDS = TILE / PER;        // lanes of a row; rows of an instruction
    const int tiles = (tokens + TILE - 1) / TILE;
    const int h = (int)(blockIdx.x % c.heads), t0 = (int)(blockIdx.x / c.heads) % tiles * TILE, b = (int)(blockIdx.x / c.heads) / tiles;
    const int n = count_of(counts, b, tokens), start = start_of(starts, b);
    const int lane = threadIdx.x, chunk = lane % LANES, first = t0 + lane / LANES;
    uint4 w[ROUNDS][2];
    int page[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = first + i * PER;
        page[i] = -1;
        if (t < n) {
            w[i][0] = stream_load(k.p + b * k.sb + t * k.st + h * k.sh + chunk * 8);
            w[i][1] = stream_load(v.p + b * v.sb + t * v.st + h * v.sh + chunk * 8);
            page[i] = page_of(c, b, start + t);
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        if (page[i] < 0) continue;
        uint8_t* const block = block_of(c, page[i], h);
        const int row = (start + first + i * PER) & (c.page - 1);
#pragma unroll
        for (int values = 0; values < 2; ++values) {
            const uint4 x = w[i][values];
            float f[8] = {bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y), bf16_lo(x.z), bf16_hi(x.z), bf16_lo(x.w), bf16_hi(x.w)};
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = f[e] == f[e] ? f[e] : 0.0f;
                amax = fmaxf(amax, fabsf(f[e]));
            }
            amax = dpp_max<0x4E>(dpp_max<0xB1>(amax));
            const int e = min(max((int)((__float_as_uint(amax) + 0x3fffffu) >> 23) - 2, 1), 252);
            *reinterpret_cast<uint32_t*>(block + idx::cache4_codes(c.page, D, values, row) + chunk * 4) = encode8(f, scale_of(e));
            if ((chunk & 3) == 0) block[idx::cache4_scales(c.page, D, values, row) + (chunk >> 2)] = (uint8_t)e;
        }
        if (c.weights && chunk == 0) c.weights[((int64_t)page[i] * c.heads + h) * c.page + row] = 0.0f;
    }
#endif
}

template <int D>
__global__ __launch_bounds__(64) void read_kernel(const Cache c, const int32_t* starts, const int32_t* counts, int tokens, uint16_t* k, uint16_t* v) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 8, PER = 64 / LANES, ROUNDS = TILE / PER;
    const int tiles = (tokens + TILE - 1) / TILE;
    const int h = (int)(blockIdx.x % c.heads), t0 = (int)(blockIdx.x / c.heads) % tiles * TILE, b = (int)(blockIdx.x / c.heads) / tiles;
    const int n = count_of(counts, b, tokens), start = start_of(starts, b);
    const int lane = threadIdx.x, chunk = lane % LANES, first = t0 + lane / LANES;
    uint32_t codes[ROUNDS][2], scales[ROUNDS][2];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = first + i * PER, page = t < n ? page_of(c, b, start + t) : -1, row = (start + t) & (c.page - 1);
        const uint8_t* const block = block_of(c, max(page, 0), h);
#pragma unroll
        for (int values = 0; values < 2; ++values) {
            codes[i][values] = scales[i][values] = 0;
            if (page >= 0) {
                codes[i][values] = *reinterpret_cast<const uint32_t*>(block + idx::cache4_codes(c.page, D, values, row) + chunk * 4);
                scales[i][values] = block[idx::cache4_scales(c.page, D, values, row) + (chunk >> 2)];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = first + i * PER;
        if (t >= tokens) break;
#pragma unroll
        for (int values = 0; values < 2; ++values)
            stream_store((values ? v : k) + (((int64_t)b * tokens + t) * c.heads + h) * D + chunk * 8, decode8(codes[i][values], scale_of(scales[i][values])));
    }
#endif
}

// order of the weights as unsigned numbers: -0 is 0, NaN the largest
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SELECT = 1024, SELECT_WAVES = SELECT / 64;       // threads, waves
constexpr int HELD = 32768;         // entries whose order stays in LDS
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

// Which entries of a (sequence, head) stay: one workgroup each.  The `heavy`-th largest weight of the old entries is found from the top, eleven bits of its
// order at a time (a histogram of those that agree so far; of the first eleven two are the weight's own, which spreads weights of a size over the bins), then
// the entries are gone through in order: those above it stay, and the first of those equal to it.  Entries of pages that the pool does not have are not there: where a
// table has such pages, entries are counted first and the recent ones placed one by one; among the old ones theirs is an order of 0, below that of every
// weight, and no more are looked for than are there.  Bound by latency: the weights are read once and
// kept in LDS, and a wave writes what stays of its own part of the entries (16 x 8 heads of up to 16384 entries, 2.9 MB of weights:
// 20 us, the longest sequence's; 8 x 8 heads of 2112 entries 9.2 us).
__global__ __launch_bounds__(SELECT) void select_kernel(const Cache c, const int32_t* lengths, int keep, int recent, int32_t* kept, int32_t* new_lengths) {
    extern __shared__ uint32_t orders[];
    __shared__ int bins[BINS], found[2], sums[2][SELECT_WAVES], missing;
    const int b = blockIdx.x / c.heads, h = blockIdx.x % c.heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = length_of(c, lengths, b), old = n - min(recent, n), pages = (n + c.page - 1) >> c.log2_page;
    int32_t* const mine = kept + ((int64_t)b * c.heads + h) * keep;
    const uint64_t below = (1ull << lane) - 1;
    const auto absent = [&](int page) { return (unsigned)c.table[b * c.table_stride + page] >= (unsigned)c.pages; };
    const int a_page = c.table[b * c.table_stride + min(tid, max(pages - 1, 0))];        // (looked at behind the weights' loads)
    for (int i = tid; i < BINS; i += SELECT) bins[i] = 0;
    if (tid == 0) missing = 0;
    __syncthreads();
    const auto any_missing = [&] {
        bool is = pages > 0 && (unsigned)a_page >= (unsigned)c.pages;
        for (int i = tid + SELECT; i < pages; i += SELECT) is |= absent(i);
        if (is) missing = 1;
        __syncthreads();
        return missing != 0;
    };
    if (n <= keep || n - old == keep) {
        if (!any_missing()) {         // all of them, or the recent ones alone
            const int stay = min(n, keep);
            if (h == 0 && tid == 0) new_lengths[b] = stay;
            for (int i = tid; i < keep; i += SELECT) mine[i] = i < stay ? n - stay + i : -1;
            return;
        }
    }
    const auto fetch = [&](int j) {
        const int page = page_of(c, b, j);
        return page < 0 ? 0u : order_of(c.weights[((int64_t)page * c.heads + h) * c.page + (j & (c.page - 1))]);
    };
    // eight entries of a thread at a time: their pages, then their weights
    const int held = min(old, HELD);
    for (int j0 = tid; j0 < held; j0 += 8 * SELECT) {
        int page[8];
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) page[i] = c.table[b * c.table_stride + (min(j0 + i * SELECT, held - 1) >> c.log2_page)];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = c.weights[((int64_t)((unsigned)page[i] < (unsigned)c.pages ? page[i] : 0) * c.heads + h) * c.page + ((j0 + i * SELECT) & (c.page - 1))];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j0 + i * SELECT < held) {
                const uint32_t u = (unsigned)page[i] < (unsigned)c.pages ? order_of(w[i]) : 0u;
                orders[j0 + i * SELECT] = u;
                atomicAdd(&bins[u >> (32 - DIGIT)], 1);
            }
    }
    const auto order = [&](int j) { return j < HELD ? orders[j] : fetch(j); };
    for (int j = HELD + tid; j < old; j += SELECT) atomicAdd(&bins[order(j) >> (32 - DIGIT)], 1);
    const bool gaps = any_missing();        // (and the first histogram is complete)
    int there = n, newest = n - old;        // entries, those of them that are recent
    if (gaps) {
        if (tid < 2) found[tid] = 0;
        __syncthreads();
        int gone = 0, gone_newest = 0;
        for (int i = tid; i < pages; i += SELECT)
            if (absent(i)) {
                const int first = i << c.log2_page, end = min(first + c.page, n);
                gone += end - first;
                gone_newest += max(end - max(first, old), 0);
            }
        atomicAdd(&found[0], gone);
        atomicAdd(&found[1], gone_newest);
        __syncthreads();
        there -= found[0];
        newest -= found[1];
    }
    const int stay = min(there, keep), heavy = stay - newest;
    if (h == 0 && tid == 0) new_lengths[b] = stay;
    for (int i = stay + tid; i < keep; i += SELECT) mine[i] = -1;
    if (gaps) {
        int place = heavy;
        for (int j0 = old; j0 < n; j0 += SELECT) {
            const bool is = j0 + tid < n && !absent((j0 + tid) >> c.log2_page);
            const uint64_t of = __ballot(is);
            __syncthreads();
            if (lane == 0) sums[0][wave] = __popcll(of);
            __syncthreads();
            int before = 0, all = 0;
            for (int w = 0; w < SELECT_WAVES; ++w) {
                before += w < wave ? sums[0][w] : 0;
                all += sums[0][w];
            }
            if (is) mine[place + before + __popcll(of & below)] = j0 + tid;
            place += all;
        }
        if (heavy == 0) return;
        __syncthreads();
    } else {
        for (int j = old + tid; j < n; j += SELECT) mine[heavy + j - old] = j;
    }
    uint32_t limit = 0;         // the heavy-th largest, as far as it is known
    int left = heavy;           // how many of those that agree with it so far are to stay
    for (int shift = 32 - DIGIT; ; shift = max(shift - DIGIT, 0)) {
        if (shift < 32 - DIGIT) {
            const int known = shift == 32 - 2 * DIGIT ? 32 - DIGIT : 32 - 2 * DIGIT;        // the bits from here on agree with the limit
            const uint32_t mask = (1u << (known - shift)) - 1;
            for (int i = tid; i < BINS; i += SELECT) bins[i] = 0;
            __syncthreads();
            for (int j = tid; j < old; j += SELECT) {
                const uint32_t u = order(j);
                if (u >> known == limit >> known) atomicAdd(&bins[u >> shift & mask], 1);
            }
            __syncthreads();
        }
        // from the largest bin on: a thread has two neighbours
        const int top = BINS - 1 - 2 * tid, x = bins[top], y = bins[top - 1];
        int upto = wave_prefix(x + y);
        if (lane == 63) sums[0][wave] = upto;
        __syncthreads();
        for (int w = 0; w < wave; ++w) upto += sums[0][w];
        const int before = upto - x - y;
        if (before < left && upto >= left) {
            const bool first = before + x >= left;
            found[0] = first ? top : top - 1;
            found[1] = left - before - (first ? 0 : x);
        }
        __syncthreads();
        limit |= (uint32_t)found[0] << shift;
        left = found[1];
        if (shift == 0) break;
    }
    // a wave's part of the entries, 64 at a time: how many are above the limit and equal to it, and then where they go
    const int part = (old + SELECT - 1) / SELECT * 64, from = min(wave * part, old), to = min(from + part, old);
    int above = 0, equal = 0;
    for (int j0 = from; j0 < to; j0 += 64) {
        const uint32_t u = j0 + lane < to ? order(j0 + lane) : 0;
        above += __popcll(__ballot(j0 + lane < to && u > limit));
        equal += __popcll(__ballot(j0 + lane < to && u == limit));
    }
    __syncthreads();
    if (lane == 0) {
        sums[0][wave] = above;
        sums[1][wave] = equal;
    }
    __syncthreads();
    above = equal = 0;
    for (int w = 0; w < wave; ++w) {
        above += sums[0][w];
        equal += sums[1][w];
    }
    for (int j0 = from; j0 < to; j0 += 64) {
        const bool in = j0 + lane < to;
        const uint32_t u = in ? order(j0 + lane) : 0;
        const uint64_t a = __ballot(in && u > limit), e = __ballot(in && u == limit);
        // in front of an entry stay those above the limit and the first `left` of the equal ones
        const int equals = equal + __popcll(e & below), place = above + __popcll(a & below) + min(equals, left);
        if (in && (u > limit || (u == limit && equals < left))) mine[place] = j0 + lane;
        above += __popcll(a);
        equal += __popcll(e);
    }
}

constexpr int MOVE = 32;        // entries per wave

// Entries to their new places.  Bound by memory: all loads of a wave's 32 entries are in flight before the first store (16 x 8 heads of 2048 entries: 67 MB
// read and written in 17 us, 4 TB/s).
template <int D>
__global__ __launch_bounds__(256) void move_kernel(const Cache c, const int32_t* kept, const int32_t* new_table, int new_pages, int64_t new_stride, int keep) {
    constexpr int LANES = D / 32, PER = 64 / LANES, ROUNDS = MOVE / PER;      // lanes of an entry's codes (16 bytes each), entries of an instruction
    const int blocks = (keep + 4 * MOVE - 1) / (4 * MOVE), lane = threadIdx.x & 63;
    const int h = (int)blockIdx.x % c.heads, i0 = ((int)(blockIdx.x / c.heads) % blocks * 4 + (threadIdx.x >> 6)) * MOVE, b = (int)(blockIdx.x / c.heads) / blocks;
    // lanes 0 .. 31 know an entry each
    const int i = i0 + (lane & (MOVE - 1)), j = i < keep ? kept[((int64_t)b * c.heads + h) * keep + i] : -1;
    const int from = page_of(c, b, j), to = i < keep && (i >> c.log2_page) < new_pages ? new_table[b * new_stride + (i >> c.log2_page)] : -1;
    const bool moves = from >= 0 && (unsigned)to < (unsigned)c.pages;
    const int r = j & (c.page - 1), s = i & (c.page - 1);
    const uint8_t* const src = block_of(c, max(from, 0), h);
    uint8_t* const dst = block_of(c, max(to, 0), h);
    v4i codes[ROUNDS][2];
    uint8_t* into[ROUNDS];
#pragma unroll
    for (int x = 0; x < ROUNDS; ++x) {
        // (every lane takes part in what it hears from the others: one that has nothing to move still knows an entry)
        const int entry = x * PER + lane / LANES, row = __shfl(r, entry, 64), new_row = __shfl(s, entry, 64), page = __shfl(from, entry, 64), new_page = __shfl(to, entry, 64);
        const bool goes = __shfl((int)moves, entry, 64);
        const uint8_t* const block = block_of(c, max(page, 0), h);
        into[x] = goes ? block_of(c, new_page, h) + new_row * (D / 2) + (lane % LANES) * 16 : nullptr;
        // (also of an entry that stays behind: a row of some page)
        codes[x][0] = *reinterpret_cast<const v4i*>(block + idx::cache4_codes(c.page, D, 0, row) + (lane % LANES) * 16);
        codes[x][1] = *reinterpret_cast<const v4i*>(block + idx::cache4_codes(c.page, D, 1, row) + (lane % LANES) * 16);
    }
    const int values = lane / MOVE;     // the lower half of the wave has the keys' scales and the weight, the upper half the values' scales
    uint32_t scales = 0;
    float weight = 0.0f;
    if (moves) {
        const uint8_t* const at = src + idx::cache4_scales(c.page, D, values, r);
        scales = D == 128 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
        if (!values) weight = c.weights[((int64_t)from * c.heads + h) * c.page + r];
    }
#pragma unroll
    for (int x = 0; x < ROUNDS; ++x)
        if (into[x]) {
            *reinterpret_cast<v4i*>(into[x]) = codes[x][0];
            *reinterpret_cast<v4i*>(into[x] + idx::cache4_codes(c.page, D, 1, 0)) = codes[x][1];
        }
    if (moves) {
        uint8_t* const at = dst + idx::cache4_scales(c.page, D, values, s);
        if (D == 128) *reinterpret_cast<uint32_t*>(at) = scales;
        else *reinterpret_cast<uint16_t*>(at) = (uint16_t)scales;
        if (!values) c.weights[((int64_t)to * c.heads + h) * c.page + s] = weight;
    }
}

int prepare_select(const char* fn) {
    static OncePerDevice once;
    const hipError_t e = raise_lds_limit(once, reinterpret_cast<const void*>(select_kernel), HELD * (int)sizeof(uint32_t));
    return e == hipSuccess ? TI8_OK : fail(TI8_ERR_HIP, "%s: cannot raise the LDS limit: %s", fn, hipGetErrorString(e));
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

int init() { return prepare_select("ti8_init"); }

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
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (c.dim == 128) hipLaunchKernelGGL(append_kernel<128>, dim3(grid), dim3(64), 0, st, c, starts, counts, (int)tokens, rk, rv);
    else hipLaunchKernelGGL(append_kernel<64>, dim3(grid), dim3(64), 0, st, c, starts, counts, (int)tokens, rk, rv);
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
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (c.dim == 128) hipLaunchKernelGGL(read_kernel<128>, dim3(grid), dim3(64), 0, st, c, starts, counts, (int)tokens, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
    else hipLaunchKernelGGL(read_kernel<64>, dim3(grid), dim3(64), 0, st, c, starts, counts, (int)tokens, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
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
    const int64_t moves = (int64_t)c.batch * c.heads * ((keep + 4 * MOVE - 1) / (4 * MOVE));
    if (moves > 0x7fffffff || (int64_t)c.batch * c.heads > 0x7fffffff) return fail(TI8_ERR_SHAPE, "%s: %lld workgroups are more than a launch takes", fn, (long long)moves);
    if (int e = prepare_select(fn)) return e;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int held = (c.capacity() < HELD ? c.capacity() : HELD) * (int)sizeof(uint32_t);
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)(c.batch * c.heads)), dim3(SELECT), held, st, c, lengths, (int)keep, (int)recent, kept, new_lengths);
    if (int e = check_launch(fn)) return e;
    if (c.dim == 128) hipLaunchKernelGGL(move_kernel<128>, dim3((unsigned)moves), dim3(256), 0, st, c, kept, new_table, (int)new_pages, new_stride, (int)keep);
    else hipLaunchKernelGGL(move_kernel<64>, dim3((unsigned)moves), dim3(256), 0, st, c, kept, new_table, (int)new_pages, new_stride, (int)keep);
    return check_launch(fn);
}
