// Attention over a cache in 4 bits.
//
// out = sum_j p_j v_j, p_j = exp(s_j - lse), s_j = scale q k_j, in one pass over the entries with a running maximum m and sum l of exp(s_j - m).  Keys and
// values go from codes to bf16 in registers (exact: a code has two significant bits and a scale is a power of two) and into
// v_mfma_f32_16x16x32_bf16 with fp32 sums; scores, m and l are fp32, probabilities are rounded to bf16 as operands of the product with the values, as
// in any attention on bf16 tensors (that rounding, 2^-9 of each, averages out over the entries; the result is rounded to bf16 anyway).
//
// step_kernel: up to 32 rows per kv head (rows = new tokens x heads that share it).  prompt_kernel: more.  weights_kernel: what every entry got.
#include <algorithm>
#include <type_traits>
#include "cache4.h"

namespace ti8 {
namespace cache4 {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef const __attribute__((address_space(4))) int32_t* constant_ints;        // read through the scalar cache

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// Exponentials are carried times 2^UP, which their common divisor takes away again: those of scores far below the maximum stay above 2^-126, below which
// v_exp_f32 gives zero, for 2^UP further (where sums are put under another maximum exp2f goes on below it).  Up to 2^(8 + UP) each (see step_kernel), their sums stay far below 2^127
constexpr float UP = 24.0f;      // (= the 24 in lse_of)
// With values below 2^63 their products' sums stay below 2^127, too (2^32 of an exponential, 2^30 entries).  A wave that comes upon a larger one (a scale of BIG or more) goes on
// with exponentials, and the sums so far, times 2^-DOWN of that, which the largest values have room for; those below 2^-86 of a row's largest then vanish.  A part in memory has
// DOWN in its maximum.
constexpr uint32_t BIG = 190;
constexpr float DOWN = 64.0f, DOWN_FACTOR = 0x1p-64f, DOWN_AWAY = 0x1p64f;

struct Args {
    Cache c;
    const int32_t *lengths, *counts;
    const uint16_t* q;
    int64_t q_sb, q_st, q_sh;
    uint16_t* out;
    float* lse;
    int2* owners;               // step_kernel: first and last workgroup of every (sequence, head)
    float* parts;               // two per workgroup, or one per row and split: see Part
    int tokens, heads, group;       // group = query heads per kv head
    float scale;
    int groups;                 // workgroups that share the units
    int blocks, block_rows, splits, shared_from;         // prompt_kernel: row blocks of a kv head, rows of each, workgroups that share its entries at most, and from how many tiles on
};

// entries of a sequence that any of its queries sees, and those that it says it has, whether or not the table has room for them
__device__ __forceinline__ int seen_of(const Args& a, int b) { return count_of(a.counts, b, a.tokens) ? length_of(a.c, a.lengths, b) : 0; }
__device__ __forceinline__ int total_of(const Args& a, int b) { return min(max(a.lengths[b], 0), 1 << 30); }

// ---- sharing out ---------------------------------------------------------------------------------------------

// What a workgroup has of the units: found by every wave from the lengths, the first 64 of which are read once
template <int UNIT, int EXTRA>     // EXTRA units of every head stand for what beginning and ending it takes
struct Lengths {
    const Args& a;
    const int lane;
    const int first, upto;      // units of a head of sequence `lane`, and of those up to it
    __device__ __forceinline__ Lengths(const Args& a_, int lane_) : a(a_), lane(lane_), first(of(lane_)), upto(wave_prefix(first)) {}
    __device__ __forceinline__ int of(int b) const { return b < a.c.batch ? idx::cache4_units(seen_of(a, b), UNIT) + EXTRA : 0; }
    __device__ __forceinline__ static int last(int v) { return __builtin_amdgcn_readlane(v, 63); }
    __device__ __forceinline__ int all() const {
        int n = last(upto);
        for (int b0 = 64; b0 < a.c.batch; b0 += 64) n += last(wave_prefix(of(b0 + lane)));
        return n * a.c.heads;
    }
    // the sequence that a unit belongs to, the units in front of that sequence and those of one of its heads
    __device__ __forceinline__ int find(int unit, int& before, int& own) const {
        int n = 0, b0 = 0, x = first, up = upto;
        while ((n + last(up)) * a.c.heads <= unit) {       // (a unit is below all(), so the walk ends with the sequences)
            n += last(up);
            b0 += 64;
            x = of(b0 + lane);
            up = wave_prefix(x);
        }
        const int here = __popcll(__ballot((n + up) * a.c.heads <= unit));        // sequences of these that end in front of the unit
        own = __builtin_amdgcn_readlane(x, here);
        before = (n + __builtin_amdgcn_readlane(up, here) - own) * a.c.heads;
        return b0 + here;
    }
};

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ v4f mfma16(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v8bf operand(uint4 x) { return __builtin_bit_cast(v8bf, x); }
// from a row's maximum, times scale log2(e), and its sum (2^UP is taken off the sum, which is exact, and not off the logarithm)
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l * 0x1p-24f)) * LN2; }
// of the four lanes that have the same place in a row of 16, in each of them
template <bool SUM>
__device__ __forceinline__ float over_rows(float x) {
    v2u y = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = SUM ? __uint_as_float(y[0]) + __uint_as_float(y[1]) : fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    y = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return SUM ? __uint_as_float(y[0]) + __uint_as_float(y[1]) : fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
#endif

// ---- few rows: a pass over the cache ---------------------------------------------------------------------------
//
// The rows of a kv head are the columns of 16 x 16 products: S^T = K Q^T with 16 entries as rows, O^T = V^T P^T with 16 elements of a head as
// rows.  So a lane has one row of queries (lane % 16) throughout, its maximum, its sum and a quarter of its result, and the probabilities
// that come out of the first product (entries 4 (lane / 16) .. + 3 of each 16) are the second one's operand as they are.
//
// A wave takes 32 entries at a time, on its own: their keys go from memory to registers in the order of the operand (a lane has 32 or 16 neighbouring
// elements of a key, which share a scale; the order of the elements in the sum is the same on both sides), their values in the same way, as
// bf16 through 32 rows of LDS that are the wave's own and out again transposed (ds_read_b64_tr_b16); values are read past the caches, which
// the keys stay in for weights_kernel (8 streams of up to 131072 entries 120 us -> 113).  The next 32 entries' loads are in flight
// meanwhile.  Four waves of a workgroup take turns and add up at the end, with their workgroups' neighbours through memory.
//
// Bound by memory where there are many entries, and nearly by the issue of instructions: 8 streams of up to 131072 entries, 616 MB, 108 to 113 us = 5.5 to 5.7 TB/s (a large copy
// here: 4.95 TB/s read and written); a SIMD issues in 0.84 of its cycles.  A step over a few thousand
// entries is mostly the kernel's beginning and end: 8 heads of 1021 entries, shared out, 6.0 us (1.5 for the launch, 1.4 to find the units, 1.3 for the
// first loads, 1.2 for the waves' sum) and 4.2 for the join.  Where tables are short every (sequence, head) is therefore left to one workgroup of eight
// waves (see step_alone): 1.5 us for 256 entries, which is how long codes take to bf16, to LDS and through two products, one after the other
// (no faster with the loads of two to four turns ahead).  Not taken: the next head's first loads in front of a head's end (registers spill,
// slower), four workgroups per CU, 64 rows in registers (see step_tiles).

template <int D>
struct Values {     // 32 rows of D bf16, 16-byte chunks permuted within a row: 16 rows' writes of a chunk and 4 x 4 rows' transposing reads spread over the banks
    static constexpr int ROW = 2 * D, BYTES = 32 * ROW;
    __device__ static __forceinline__ int swizzle(int row) {
        return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
};

template <int D>
struct Part {       // what a workgroup leaves of a (sequence, head) that it has not got alone: unnormalised results, maxima (times scale log2(e)) and sums of its rows
    static constexpr int ROW = D + 4;       // (16-byte aligned)
};

constexpr int WAVES = 4, ENTRIES = 32;      // waves of a workgroup; entries of a wave's turn
// Units that beginning and ending a head count for when the units are shared out: 16 sequences of 1 to 4096 entries, 32 heads each: 37.5 us with none, 28.6
// with two, 30.9 with four, 32.4 with six
constexpr int EXTRA = 2;
static_assert(idx::CACHE4_UNIT == WAVES * ENTRIES, "a unit is a turn of every wave");

template <int D, int TILES, bool OWN>     // TILES * 16 rows; whether every (sequence, head) has a workgroup of its own, of twice the waves
__global__ __launch_bounds__(OWN ? 2 * WAVES * 64 : WAVES * 64, OWN || TILES == 2 ? 2 : 3) void step_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using V = Values<D>;
    constexpr int STEPS = D / 32;       // words of codes of an entry that a lane has; products over D
    constexpr int BLOCKS = D / 16, NW = OWN ? 2 * WAVES : WAVES;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[NW * V::BYTES];
    __shared__ float stats[NW][2][16];
    const Cache& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, quarter = lane >> 4;
    idx::Share share;
    int b, h, total, length, per_head, end, left, unit = 0;
    const auto read_length = [&] {
        total = __builtin_amdgcn_readfirstlane(total_of(a, b));
        length = __builtin_amdgcn_readfirstlane(count_of(a.counts, b, a.tokens)) ? min(total, c.capacity()) : 0;
    };
    if constexpr (OWN) {
        b = blockIdx.x / c.heads;
        h = blockIdx.x % c.heads;
        read_length();
        per_head = idx::cache4_units(length, NW * ENTRIES);
        end = left = per_head + EXTRA;
    } else {
        const Lengths<idx::CACHE4_UNIT, EXTRA> lengths(a, lane);
        share = idx::share_out(lengths.all(), a.groups);
        if ((int)blockIdx.x >= share.groups) return;
        const int begin = idx::share_begin(share, blockIdx.x);
        int before;
        end = idx::share_begin(share, blockIdx.x + 1);
        b = lengths.find(begin, before, per_head);
        read_length();
        const int at_begin = (begin - before) % per_head;
        h = (begin - before) / per_head;
        unit = max(at_begin - EXTRA, 0);
        left = end - begin - max(EXTRA - at_begin, 0);
        per_head -= EXTRA;
    }
    uint8_t* const mine = smem + wave * V::BYTES;
    // (a negative scale: the queries' signs are changed, which is exact.  Above zero, so that what is masked stays at -inf)
    const float factor = fmaxf(fabsf(a.scale) * LOG2E, 0x1p-126f);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;

    while (left > 0) {
        const int n = min(left, per_head - unit), first = unit * NW + wave, last = (unit + n) * NW;       // this wave's turns
        const int count = count_of(a.counts, b, a.tokens), rows = count * a.group, older = total - count;
        const constant_ints table = (constant_ints)(c.table + b * c.table_stride);
        struct Turn {
            uint32_t k[2][STEPS], v[2][STEPS], ks[2], vs[2];
            int absent;     // a bit for each 16 whose page the pool does not have
        };
        const auto pages_of = [&](int turn, int (&page)[2]) {
#pragma unroll
            for (int u = 0; u < 2; ++u) page[u] = table[min(turn * ENTRIES + u * 16, c.capacity() - 1) >> c.log2_page];
        };
        const auto load = [&](int turn, const int (&page)[2], Turn& x) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = turn * ENTRIES + u * 16;
                const bool there = j < length && (unsigned)page[u] < (unsigned)c.pages;
                const uint8_t* const block = block_of(c, there ? page[u] : 0, h);
                const int row = (j & (c.page - 1)) + r16;
                const uint8_t *const kc = block + idx::cache4_codes(c.page, D, 0, row) + quarter * (D / 8), *const vc = block + idx::cache4_codes(c.page, D, 1, row) + quarter * (D / 8);
                if constexpr (D == 128) {
                    const uint4 y = *reinterpret_cast<const uint4*>(kc), z = stream_load(vc);
                    x.k[u][0] = y.x; x.k[u][1] = y.y; x.k[u][2] = y.z; x.k[u][3] = y.w;
                    x.v[u][0] = z.x; x.v[u][1] = z.y; x.v[u][2] = z.z; x.v[u][3] = z.w;
                } else {
                    const uint2 y = *reinterpret_cast<const uint2*>(kc);
                    const v2i z = __builtin_nontemporal_load(reinterpret_cast<const v2i*>(vc));
                    x.k[u][0] = y.x; x.k[u][1] = y.y;
                    x.v[u][0] = z[0]; x.v[u][1] = z[1];
                }
                x.ks[u] = block[idx::cache4_scales(c.page, D, 0, row) + quarter * (D / 4) / GROUP];
                x.vs[u] = block[idx::cache4_scales(c.page, D, 1, row) + quarter * (D / 4) / GROUP];
                // (entries that are not there: whatever lies in their place must not be multiplied by a probability of zero)
                if (!there || j + r16 >= length) x.vs[u] = 0;
            }
            const int j = turn * ENTRIES;
            const bool one = (unsigned)page[0] < (unsigned)c.pages, two = (unsigned)page[1] < (unsigned)c.pages;
            x.absent = (one || j >= length ? 0 : 1) | (two || j + 16 >= length ? 0 : 2);
        };

        Turn now;
        int page[2];
        pages_of(first, page);
        if (first < last) load(first, page, now);
        pages_of(min(first + NW, last - 1), page);

        // this wave's queries as operands, and up to where each row sees
        v8bf q[TILES][STEPS];
        int sees[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int row = t * 16 + r16, token = row / a.group, head = h * a.group + row % a.group;
            sees[t] = row < rows ? min(older + token + 1, length) : 0;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (row < rows) x = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + token * a.q_st + head * a.q_sh + quarter * (D / 4) + s * 8);
                q[t][s] = operand(make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip));
            }
        }
        const int all_see = min(older + 1, length);         // entries that every row sees

        v4f o[TILES][BLOCKS];
        float top[TILES], shift[TILES], sum[TILES];      // maximum, what is taken from a score times factor, sum of this lane's entries
        float up = UP;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            top[t] = -INFINITY;
            shift[t] = sum[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) o[t][d] = v4f{0, 0, 0, 0};
        }

        const auto compute = [&](int turn, const Turn& x) {
            v4f s[TILES][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float scale = scale_of(x.ks[u]);
#pragma unroll
                for (int t = 0; t < TILES; ++t) s[t][u] = v4f{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const v8bf k = operand(decode8(x.k[u][i], scale));
#pragma unroll
                    for (int t = 0; t < TILES; ++t) s[t][u] = mfma16(k, q[t][i], s[t][u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float scale = scale_of(x.vs[u]);
                const int row = u * 16 + r16;
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
                    *reinterpret_cast<uint4*>(mine + row * V::ROW + (((quarter * STEPS + i) ^ V::swizzle(row)) << 4)) = decode8(x.v[u][i], scale);
            }
            const int j0 = turn * ENTRIES;
            const bool big = __any(max(x.vs[0], x.vs[1]) >= BIG);
            if (j0 + ENTRIES > all_see || x.absent || big) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (j0 + u * 16 + quarter * 4 + i >= sees[t] || (x.absent >> u & 1)) s[t][u][i] = -INFINITY;
                if (big && up == UP) {
                    up -= DOWN;
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        shift[t] += DOWN;
                        sum[t] *= DOWN_FACTOR;
#pragma unroll
                        for (int d = 0; d < BLOCKS; ++d) o[t][d] *= DOWN_FACTOR;
                    }
                }
            }
            v8bf p[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const v4f z = s[t][0], y = s[t][1];
                const float largest = over_rows<false>(fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))));
                // sums go on under the old maximum until a score is 2^8 above it: the same result, as everything is divided by the sum in the end
                if (__any((largest - top[t]) * factor > 8.0f)) {
                    const float higher = fmaxf(top[t], largest), shrink = higher == -INFINITY ? 1.0f : exp2f((top[t] - higher) * factor);
                    top[t] = higher;
                    shift[t] = higher == -INFINITY ? 0.0f : higher * factor - up;
                    sum[t] *= shrink;
#pragma unroll
                    for (int d = 0; d < BLOCKS; ++d) o[t][d] *= shrink;
                }
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][i & 3], factor, -shift[t]));
                sum[t] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                p[t] = operand(make_uint4(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]), pack_bf16x2(e[6], e[7])));
            }
            // (LDS is read back by the wave that wrote it, which its LDS instructions' order is enough for)
            asm volatile("" ::: "memory");
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) {
                const int row = quarter * 4 + (r16 >> 2), chunk = d * 2 + ((r16 >> 1) & 1);
                const uint8_t* const at = mine + row * V::ROW + ((chunk ^ V::swizzle(row)) << 4) + (r16 & 1) * 8;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 16 * V::ROW));
                const v8bf v = __builtin_bit_cast(v8bf, (v8s)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int t = 0; t < TILES; ++t) o[t][d] = mfma16(v, p[t], o[t][d]);
            }
            asm volatile("" ::: "memory");
        };

        for (int turn = first; turn < last; turn += NW) {
            Turn next;
            if (turn + NW < last) load(turn + NW, page, next);
            pages_of(min(turn + 2 * NW, last - 1), page);
            compute(turn, now);
            now = next;
        }

        // the waves' results meet in LDS, 16 rows at a time
        const bool whole = OWN || n == per_head;
        if (!OWN && unit == 0 && threadIdx.x == 0) a.owners[b * c.heads + h] = make_int2(blockIdx.x, whole ? blockIdx.x : idx::share_of(share, end - left + per_head - 1));
        float* const part = a.parts + ((int64_t)blockIdx.x * 2 + (unit == 0)) * (TILES * 16) * Part<D>::ROW;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const float total = over_rows<true>(sum[t]);
            __syncthreads();
            if (quarter == 0) {
                stats[wave][0][r16] = top[t];
                stats[wave][1][r16] = up == UP ? total : -total;      // (the sign says how they are carried)
            }
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
                *reinterpret_cast<v4f*>(mine + r16 * (4 * D) + (((d * 4 + quarter) ^ r16) << 4)) = o[t][d];
            __syncthreads();
            const int row = threadIdx.x / (NW * 4), lane_of = threadIdx.x % (NW * 4);
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, stats[w][0][row]);
            float f[NW];
            bool down = false;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                f[w] = stats[w][0][row] == -INFINITY ? 0.0f : exp2f((stats[w][0][row] - m) * factor);
                down |= stats[w][1][row] < 0.0f;
            }
            if (__any(down))
#pragma unroll
                for (int w = 0; w < NW; ++w) f[w] *= down && !(stats[w][1][row] < 0.0f) ? DOWN_FACTOR : 1.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w)        // (a NaN in the sum passes a maximum of -inf)
                l += stats[w][0][row] == -INFINITY ? stats[w][1][row] : fabsf(stats[w][1][row]) * f[w];
            const int at = t * 16 + row, token = at / a.group;
            if (at >= rows) l = 0.0f;       // (no query: zeros were multiplied)
            const int64_t to = ((int64_t)b * a.tokens + token) * a.heads + h * a.group + at % a.group;
            const float norm = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int i = 0; i < (D + NW * 16 - 1) / (NW * 16); ++i) {
                const int chunk = i * (NW * 4) + lane_of;
                if (chunk >= D / 4) break;
                v4f x{0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; ++w) x += *reinterpret_cast<const v4f*>(smem + w * V::BYTES + row * (4 * D) + ((chunk ^ row) << 4)) * f[w];
                if (!whole) {
                    if (at < rows) *reinterpret_cast<v4f*>(part + at * Part<D>::ROW + chunk * 4) = x;
                } else if (at < a.tokens * a.group)
                    *reinterpret_cast<uint2*>(a.out + to * D + chunk * 4) = make_uint2(pack_bf16x2(x[0] * norm, x[1] * norm), pack_bf16x2(x[2] * norm, x[3] * norm));
            }
            if (lane_of == 0) {
                if (!whole) {
                    if (at < rows) *reinterpret_cast<float2*>(part + at * Part<D>::ROW + D) = make_float2(m * factor + (down ? DOWN : 0.0f), l);
                } else if (at < a.tokens * a.group) a.lse[to] = lse_of(m * factor, down ? l * DOWN_AWAY : l);
            }
        }
        left -= n + EXTRA;
        unit = 0;
        if (++h == c.heads && left > 0) {
            h = 0;
            ++b;
            read_length();
            per_head = idx::cache4_units(length, idx::CACHE4_UNIT);
        }
        __syncthreads();        // nobody writes values while somebody still adds up
    }
#endif
}

// A row from its `n` parts: the first one, and the others behind `rest` at a distance.  GROUPS times D / 4 lanes share it (with 256 threads of a workgroup in
// all); the largest maximum comes first, so that the parts themselves are independent loads.
template <int D, int GROUPS>
__device__ __forceinline__ void join(const Args& a, const float* one, const float* rest, int64_t distance, int n, int64_t row, bool is) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LANES = D / 4, THREADS = GROUPS * LANES;
    __shared__ v4f shared[GROUPS][LANES];
    __shared__ float shared_m[GROUPS], shared_l[GROUPS];
    const int tid = threadIdx.x % THREADS, group = tid / LANES, at = tid % LANES;
    const auto part = [&](int i) { return i ? rest + i * distance : one; };
    float m = -INFINITY, l = 0.0f;
    for (int i = tid; i < n; i += THREADS) m = fmaxf(m, part(i)[D]);
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (GROUPS > 1) {
        if (at == 0) shared_m[group] = m;
        __syncthreads();
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) m = fmaxf(m, shared_m[g]);
    }
    // (a NaN in a sum passes a maximum of -inf)
    const auto weight = [&](float pm) { return pm == -INFINITY ? 0.0f : exp2f(pm - m); };
    for (int i = tid; i < n; i += THREADS) {
        const float pm = part(i)[D], pl = part(i)[D + 1];
        l += pm == -INFINITY ? pl : pl * weight(pm);
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) l += __shfl_xor(l, d, 64);
    v4f o{0, 0, 0, 0};
#pragma unroll 4
    for (int i = group; i < n; i += GROUPS) o += *reinterpret_cast<const v4f*>(part(i) + at * 4) * weight(part(i)[D]);
    if (GROUPS > 1) {
        shared[group][at] = o;
        if (at == 0) shared_l[group] = l;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) {
            o += shared[g][at];
            l += shared_l[g];
        }
    }
    if (!is) {      // no query, and no parts
        l = 0.0f;
        o = v4f{0, 0, 0, 0};
    }
    const float norm = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(a.out + row * D + at * 4) = make_uint2(pack_bf16x2(o[0] * norm, o[1] * norm), pack_bf16x2(o[2] * norm, o[3] * norm));
    if (at == 0) a.lse[row] = lse_of(m, l);
#endif
}

// Rows whose (sequence, head) several workgroups had: one workgroup each.  Bound by latency (owners, maxima, parts, one after the other): 3.8 to 5 us
template <int D, int TILES>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const Cache& c = a.c;
    const int rows = a.tokens * a.group, row = blockIdx.x % rows, h = (int)(blockIdx.x / rows) % c.heads, b = (int)(blockIdx.x / rows) / c.heads;
    const int2 owners = a.owners[b * c.heads + h];
    const int first = owners.x, last = owners.y;
    if (first == last) return;
    // a workgroup's second part is the one that starts with a head's first unit: here that of the first workgroup
    constexpr int64_t PART = TILES * 16 * Part<D>::ROW;
    const float* const from = a.parts + first * 2 * PART + row * Part<D>::ROW;
    join<D, 1024 / D>(a, from + PART, from, 2 * PART, last - first + 1, ((int64_t)b * a.tokens + row / a.group) * a.heads + h * a.group + row % a.group,
                      row / a.group < count_of(a.counts, b, a.tokens));
#endif
}

// ---- many rows: prompts ------------------------------------------------------------------------------------------
//
// A wave has 32 rows of queries as the columns of 32 x 32 products (S^T = K Q^T, O^T = V^T P^T: a lane has one row of queries, as above); the waves
// of a workgroup go through the entries together, 64 at a time, which they turn into bf16 in LDS once for all, two tiles ahead (one, where a
// workgroup of four waves shares a CU with others); the codes of the tile behind that are on their way meanwhile.
// A wave's scores of 32 entries are multiplied while it takes the exponentials of the 32 before, and the maxima of the one's are found while the other's
// values are multiplied: products and vector instructions of a wave alternate, or they would take turns on all waves, which the tiles keep in step.
// A head's row blocks lie on one XCD, whose L2 then serves the entries; where there are too few row blocks for the chip, several workgroups share the
// entries of one and join_rows_kernel adds them up.
//
// 2 x 2048 tokens of 32 heads behind 6144 entries 462 to 472 us = 1.02 to 1.04 PFLOP/s (a matrix product of the library: 1.4 to 1.46).  No unit is full: of the cycles the
// matrix pipe has 0.42, the vector unit 0.44 (half of the former's beside the latter: 0.65 together), LDS 0.53, of which half are bank conflicts; waves
// wait 0.37 of their time.  Short prompts of several lengths: bound by the longest row block's
// chain of tiles (2 us each with 256 rows).

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int TILE = 64;        // entries of a tile

template <int D>
struct Tile32 {     // rows of D bf16 in LDS, 32 bytes apart: neighbouring rows' chunks fall into other banks, and addresses are sums, most of them constants
    static constexpr int ROW = 2 * D + 32, BYTES = TILE * ROW;
    // this lane's chunk of an operand whose rows are the tile's: plus 32 per step, 32 ROW per 32 rows
    __device__ static __forceinline__ int rows_at(int lane) { return (lane & 31) * ROW + (lane >> 5) * 16; }
    // the same of an operand over the rows (transposing read): plus 64 per column tile, 8 ROW per 8 rows
    __device__ static __forceinline__ int columns_at(int lane) {
        const int i = lane & 15;
        return (4 * (lane >> 5) + (i >> 2)) * ROW + ((lane >> 4) & 1) * 32 + (i & 3) * 8;
    }
};

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ v16f mfma32(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
template <bool SUM>
__device__ __forceinline__ float over_halves(float x) {
    const v2u y = __builtin_bit_cast(v2u, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return SUM ? __uint_as_float(y[0]) + __uint_as_float(y[1]) : fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
// 16 or 8 bytes of codes of an entry and the scale of their elements
template <int D>
struct Codes {
    static constexpr int WORDS = D / 32;
    uint32_t w[WORDS], scale;
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales) {
        if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(codes);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(codes);
            w[0] = x.x; w[1] = x.y;
        }
        scale = *scales;
    }
};
#endif

// tiles in LDS: three with eight waves, which have a CU to themselves
template <int NW> constexpr int PROMPT_STAGES = NW == 8 ? 3 : 2;

// What the rows from `row0` on, a block, of a sequence see: tiles of entries, and how many workgroups share them (the others of a.splits have nothing to do).
// One leaves no parts.
struct BlockSees {
    int most, tiles, parts;
    __device__ __forceinline__ BlockSees(const Args& a, int row0, int count, int older, int length) {
        const int rows = count * a.group;
        most = row0 < rows ? max(min(older + (min(row0 + a.block_rows, rows) - 1) / a.group + 1, length), 0) : 0;
        tiles = (most + TILE - 1) / TILE;
        parts = tiles < a.shared_from ? 1 : min(a.splits, (tiles + 3) / 4);
    }
};

// NW waves, of which SHARES at a time have the same 32 rows: with two, each takes its own half of every tile, and they add up at the end
template <int D, int NW, int SHARES>
__global__ __launch_bounds__(NW * 64, 2) void prompt_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = Tile32<D>;
    constexpr int STEPS = D / 16, BLOCKS = D / 32, PARTS = 8 / NW;      // PARTS: of a tile (keys and values in quarters) that a wave converts
    constexpr int STAGES = PROMPT_STAGES<NW>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];        // [STAGES][keys, values]
    __shared__ __attribute__((aligned(16))) int absent[STAGES][4];        // whether the pool does not have the page of 16 entries of a tile
    __shared__ int any_big;     // whether some values so far have a scale of BIG or more
    const Cache& c = a.c;
    const idx::AttentionPlace place = idx::cache4_place(blockIdx.x, c.batch * c.heads, a.blocks * a.splits);
    if (place.pair >= c.batch * c.heads) return;
    const int b = place.pair / c.heads, h = place.pair % c.heads;
    const int block = place.block / a.splits, split = place.block % a.splits;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, half = lane >> 5, r16 = lane & 15, quarter = lane >> 4;
    constexpr int ROWS_OF = NW / SHARES * 32;
    const int mine_of = wave / (NW / SHARES);      // which half of a tile, with two shares
    const int count = count_of(a.counts, b, a.tokens), length = length_of(c, a.lengths, b), older = total_of(a, b) - count, rows = count * a.group;
    const int row0 = block * ROWS_OF, row = row0 + wave % (NW / SHARES) * 32 + r32;
    // entries that this lane's row, any row of the workgroup and any row of the wave sees
    const auto sees_of = [&](int r) { return max(min(older + r / a.group + 1, length), 0); };
    const int sees = row < rows ? sees_of(row) : 0;
    const BlockSees block_sees(a, row0, count, older, length);
    if (split >= block_sees.parts) return;
    const int wave0 = row0 + wave % (NW / SHARES) * 32, wave_most = wave0 < rows ? sees_of(min(wave0 + 32, rows) - 1) : 0;
    const int tiles = block_sees.tiles, begin = (int)((int64_t)split * tiles / block_sees.parts), end = (int)((int64_t)(split + 1) * tiles / block_sees.parts);
    if (threadIdx.x == 0) any_big = 0;
    // entries that every row of the workgroup sees: none where the pool does not have all the pages
    bool gaps = false;
    for (int i = (begin * TILE >> c.log2_page) + threadIdx.x; i < (min(end * TILE, length) + c.page - 1) >> c.log2_page; i += NW * 64)
        gaps |= (unsigned)c.table[b * c.table_stride + i] >= (unsigned)c.pages;
    const int all = !__syncthreads_or(gaps) && row0 < rows ? sees_of(row0) : 0;
    const float factor = fmaxf(fabsf(a.scale) * LOG2E, 0x1p-126f);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    const constant_ints table = (constant_ints)(c.table + b * c.table_stride);

    v8bf q[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row < rows) x = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (row / a.group) * a.q_st + (h * a.group + row % a.group) * a.q_sh + s * 16 + half * 8);
        q[s] = operand(make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip));
    }
    v16f o[BLOCKS];
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float top = -INFINITY, shift = 0.0f, sum = 0.0f, up = UP;

    Codes<D> raw[PARTS];
    int there[PARTS];
    // the wave's part p of a tile: keys (p < 4) or values of 16 entries; a lane has a quarter of an entry's elements
    const auto load = [&](int tile) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int p = wave + i * NW, j = tile * TILE + (p & 3) * 16;
            const int page = table[min(j, c.capacity() - 1) >> c.log2_page];
            there[i] = j < length && (unsigned)page < (unsigned)c.pages;
            const uint8_t* const from = block_of(c, there[i] ? page : 0, h);
            const int at = (j & (c.page - 1)) + r16;
            raw[i].load(from + idx::cache4_codes(c.page, D, p >> 2, at) + quarter * (D / 8), from + idx::cache4_scales(c.page, D, p >> 2, at) + quarter * (D / 4) / GROUP);
            if (!there[i] || j + r16 >= length) raw[i].scale = 0;       // (nothing that is no number)
        }
    };
    const auto convert = [&](int tile, int stage) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int p = wave + i * NW, at = (p & 3) * 16 + r16;
            uint8_t* const to = smem + (stage * 2 + (p >> 2)) * T::BYTES + at * T::ROW;
            if (p >= 4 && __any(raw[i].scale >= BIG)) any_big = 1;
            const float scale = scale_of(raw[i].scale);
#pragma unroll
            for (int w = 0; w < Codes<D>::WORDS; ++w)
                *reinterpret_cast<uint4*>(to + (quarter * Codes<D>::WORDS + w) * 16) = decode8(raw[i].w[w], scale);
            if (p < 4 && lane == 0) absent[stage][p] = !there[i] && tile * TILE + p * 16 < length;
        }
    };
    const int rows_at = T::rows_at(lane), columns_at = T::columns_at(lane);
    // scores of half `u` of a tile
    const auto scores = [&](int stage, int u) {
        const uint8_t* const kt = smem + rows_at + stage * 2 * T::BYTES;
        v16f s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < STEPS; ++x) s = mfma32(*reinterpret_cast<const v8bf*>(kt + u * 32 * T::ROW + x * 32), q[x], s);
        return s;
    };
    const auto gone_of = [&](int stage) {       // a bit for each 16 entries whose page the pool does not have
        const v4i x = *reinterpret_cast<const v4i*>(absent[stage]);
        return __builtin_amdgcn_readfirstlane(x[0] | x[1] << 1 | x[2] << 2 | x[3] << 3);
    };
    // -inf for entries that the row does not see
    const auto mask = [&](v16f& s, int tile, int u, int gone) {
        const int up_to = sees - (tile * TILE + u * 32) - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (8 * (i >> 2) + (i & 3) >= up_to || (gone >> (2 * u + (i >> 3)) & 1)) s[i] = -INFINITY;
    };
    const auto largest_of = [&](const v16f& s) {
        // (v_med3_f32 with infinity is a maximum that does not ask whether its operands are quiet)
        float m = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) m = __builtin_amdgcn_fmed3f(m, s[i], INFINITY);
        return over_halves<false>(m);
    };
    const auto raise = [&](float largest, int big) {
        if (__any((largest - top) * factor > 8.0f || big)) {       // see step_kernel
            const float higher = fmaxf(top, largest);
            float shrink = higher == -INFINITY ? 1.0f : exp2f((top - higher) * factor);
            if (__any(big) && up == UP) {
                up -= DOWN;
                shrink *= DOWN_FACTOR;
            }
            top = higher;
            shift = higher == -INFINITY ? 0.0f : higher * factor - up;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) o[d] *= shrink;
        }
    };
    const auto exponentials = [&](v16f& s, v8bf (&p)[2]) {
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], factor, -shift));
            part[i & 3] += s[i];
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
            p[x] = operand(make_uint4(pack_bf16x2(s[8 * x], s[8 * x + 1]), pack_bf16x2(s[8 * x + 2], s[8 * x + 3]),
                                      pack_bf16x2(s[8 * x + 4], s[8 * x + 5]), pack_bf16x2(s[8 * x + 6], s[8 * x + 7])));
    };
    const auto add_values = [&](int stage, int u, const v8bf (&p)[2]) {
        const uint8_t* const vt = smem + columns_at + (stage * 2 + 1) * T::BYTES;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d) {
                const uint8_t* const at = vt + (u * 32 + x * 16) * T::ROW + d * 64;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 8 * T::ROW));
                o[d] = mfma32(__builtin_bit_cast(v8bf, (v8s)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), p[x], o[d]);
            }
    };
    // from the scores of a half tile (s) to the next one's, of half u of a tile in `ahead`; the values are half `of` of `stage`
    v16f s;
    // (with `last` they are those of the next tile, and the first multiplied by its values)
    const auto step = [&](int stage, int of, int ahead, int u, int tile, int gone, auto masked, auto last) {
        v8bf p[2];
        const int big = last ? any_big : 0;     // (the next tile was converted before the waves last met)
        v16f other = scores(ahead, u);
        exponentials(s, p);
        if (masked) mask(other, tile, u, gone);
        const float largest = largest_of(other);
        add_values(stage, of, p);
        s = other;
        raise(largest, big);
    };

    if (begin < end) {
        const int mine = min(end, (wave_most + TILE - 1) / TILE);       // this wave's tiles end here
        load(begin);
        convert(begin, 0);
        if (begin + 1 < end) load(begin + 1);
        if (STAGES == 3) {
            if (begin + 1 < end) convert(begin + 1, 1);
            if (begin + 2 < end) load(begin + 2);
        }
        __syncthreads();
        if (begin < mine) {
            s = scores(0, SHARES == 2 ? mine_of : 0);
            mask(s, begin, SHARES == 2 ? mine_of : 0, gone_of(0));
            raise(largest_of(s), __builtin_amdgcn_readfirstlane(any_big));
        }
        int stage = 0;
        const auto walk = [&](int from, int to, auto masked) {
            for (int tile = from; tile < to; ++tile) {
                const int next = stage + 1 == STAGES ? 0 : stage + 1;
                if (tile > begin) __syncthreads();      // nobody reads the tile before; with three stages the next one is there
                const int into = STAGES == 3 ? (next + 1 == STAGES ? 0 : next + 1) : next, ready = tile + STAGES - 1;
                if (ready < end) convert(ready, into);
                if (ready + 1 < end) load(ready + 1);
                if (SHARES == 1 && tile < mine) step(stage, 0, stage, 1, tile, masked ? gone_of(stage) : 0, masked, std::false_type{});
                if (STAGES == 2) __syncthreads();       // the next tile is there
                const int of = SHARES == 2 ? mine_of : 1, u = SHARES == 2 ? mine_of : 0;
                if (tile + 1 < mine) step(stage, of, next, u, tile + 1, masked ? gone_of(next) : 0, masked, std::true_type{});
                else if (tile < mine) {
                    v8bf p[2];
                    exponentials(s, p);
                    add_values(stage, of, p);
                }
                stage = next;
            }
        };
        // up to here every row sees every entry of a tile and of the next one
        const int clear = min(max(all / TILE - 1, begin), end);
        walk(begin, clear, std::false_type{});
        walk(clear, end, std::true_type{});
        raise(-INFINITY, __builtin_amdgcn_readfirstlane(any_big));        // (a wave whose rows see none of the last tiles: all waves carry alike)
    }
    sum = over_halves<true>(sum);
    if constexpr (SHARES == 2) {
        __syncthreads();
        float* const meet = reinterpret_cast<float*>(smem) + (wave % (NW / 2)) * (BLOCKS * 16 + 2) * 64 + lane;
        if (mine_of == 1) {
#pragma unroll
            for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) meet[(d * 16 + i) * 64] = o[d][i];
            meet[BLOCKS * 16 * 64] = top;
            meet[(BLOCKS * 16 + 1) * 64] = sum;
        }
        __syncthreads();
        if (mine_of == 1) return;
        const float other = meet[BLOCKS * 16 * 64], more = meet[(BLOCKS * 16 + 1) * 64], higher = fmaxf(top, other);
        const float fa = top == -INFINITY ? 0.0f : exp2f((top - higher) * factor), fb = other == -INFINITY ? 0.0f : exp2f((other - higher) * factor);
        sum = (top == -INFINITY ? sum : sum * fa) + (other == -INFINITY ? more : more * fb);        // (a NaN in a sum passes a maximum of -inf)
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * fa + meet[(d * 16 + i) * 64] * fb;
        top = higher;
    }
    // (the row is found anew, from the lane: kept in registers it would be spilled)
    int lane_of = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane_of));
    const int half_of = lane_of >> 5, row_of = row0 + wave % (NW / SHARES) * 32 + (lane_of & 31), token = row_of / a.group, head = h * a.group + row_of % a.group;
    if (token >= a.tokens) return;
    const int64_t to = ((int64_t)b * a.tokens + token) * a.heads + head;
    if (block_sees.parts > 1) {
        float* const part = a.parts + (to * a.splits + split) * Part<D>::ROW;
#pragma unroll
        for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<v4f*>(part + d * 32 + 2 * i + 4 * half_of) = v4f{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (half_of == 0) {
            part[D] = top * factor + (UP - up);
            part[D + 1] = row_of < rows ? sum : 0.0f;
        }
        return;
    }
    if (row_of >= rows) sum = 0.0f;
    const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint2*>(a.out + to * D + d * 32 + 2 * i + 4 * half_of) = make_uint2(pack_bf16x2(o[d][i] * norm, o[d][i + 1] * norm), pack_bf16x2(o[d][i + 2] * norm, o[d][i + 3] * norm));
    if (half_of == 0) a.lse[to] = lse_of(top * factor, up == UP ? sum : sum * DOWN_AWAY);
#endif
}

// Rows whose entries several workgroups shared.  Bound by memory, or by latency where there are few
template <int D, int GROUPS>
__global__ __launch_bounds__(256) void join_rows_kernel(const Args a, int64_t rows) {
    const int64_t row = (int64_t)blockIdx.x * (1024 / D / GROUPS) + threadIdx.x / (GROUPS * D / 4);
    if (row >= rows) return;
    const uint32_t token_of = (uint32_t)row / (uint32_t)a.heads, b = token_of / (uint32_t)a.tokens;      // (fewer than 2^31 rows: ti8_cache4_attention)
    const int at = (int)(token_of % (uint32_t)a.tokens) * a.group + (int)((uint32_t)row % (uint32_t)a.heads) % a.group;
    const int count = count_of(a.counts, b, a.tokens);
    const int parts = BlockSees(a, at / a.block_rows * a.block_rows, count, total_of(a, b) - count, length_of(a.c, a.lengths, b)).parts;
    if (parts == 1) return;
    const float* const from = a.parts + row * a.splits * Part<D>::ROW;
    join<D, GROUPS>(a, from, from, Part<D>::ROW, parts, row, true);
}

// ---- what the entries got ------------------------------------------------------------------------------------------
//
// weights of entry j += sum over rows of exp(s_j - lse): the scores once more, with the entries as columns of 32 x 32 products, so that a lane adds up the
// rows of one entry.  Units of 256 entries are shared out as for step_kernel; each of eight waves has the keys of 32 in registers and goes through the rows
// that see them, which the workgroup brings into LDS 64 at a time, two tiles ahead, without a trip through registers.  An entry of a sequence has one owner, which adds
// its rows up in a fixed order; the sum goes to the weight as an atomic addition, because sequences with a common beginning may share its pages (then
// the order of their additions is open, otherwise a weight gets one).
//
// Few rows: bound by the beginning and by memory (32 streams of 2048 entries of 8 heads: 39 MB in 15 us); many: by the issue of a SIMD, 0.87 of its cycles (8 x 1024 tokens
// over 4096 entries of 32 heads: 315 us = 0.76 PFLOP/s), and, with one or two units per workgroup, by the units that most rows see.  The loads to LDS
// are global_load_lds: in front of every read of LDS the compiler waits for all buffer loads to LDS, also for those two tiles ahead (390 us).
// Not taken: a step's exponentials beside the next scores' products in one wave (354 us: the waves of a SIMD overlap as it is, and registers are short);
// lse from the attention's parts instead of the joined one, which would save a launch's 4 us but reads all parts of a head in every workgroup.

constexpr int COLUMNS = 32, WEIGHT_WAVES = 8, WEIGHTS_UNIT = WEIGHT_WAVES * COLUMNS, ROWS = 64, RING = 3;

#if defined(__HIP_DEVICE_COMPILE__)
// all but this wave's last N loads have landed, its LDS reads have returned, and the same holds for the other waves
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 0xf) | ((N >> 4) << 14) | 0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
#endif

template <int D>
__global__ __launch_bounds__(WEIGHT_WAVES * 64, 4) void weights_kernel(const Args a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int UNIT = WEIGHTS_UNIT, STEPS = D / 16, ROW = 2 * D, CHUNKS = D / 8, PASSES = ROWS * CHUNKS / (WEIGHT_WAVES * 64), LOADS = PASSES + 1;
    __shared__ __attribute__((aligned(1024))) int8_t smem[RING * (ROWS * ROW + WEIGHT_WAVES * ROWS * 4)];
    const auto queries = [&](int stage) { return smem + stage * (ROWS * ROW); };
    // times log2(e) once they are there; every wave has its own
    const auto lses = [&](int stage) { return reinterpret_cast<float*>(smem + RING * ROWS * ROW + (stage * WEIGHT_WAVES + (int)(threadIdx.x >> 6)) * (ROWS * 4)); };
    const Cache& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, half = lane >> 5;
    const Lengths<UNIT, 0> lengths(a, lane);
    const idx::Share share = idx::share_out(lengths.all(), a.groups);
    if ((int)blockIdx.x >= share.groups) return;
    const int begin = idx::share_begin(share, blockIdx.x), end = idx::share_begin(share, blockIdx.x + 1);
    const float factor = fabsf(a.scale) * LOG2E;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    const int step_token = ROWS / a.group, step_head = ROWS % a.group;
    struct Unit {
        int b, h, unit, length, count, older, per_head;
        __device__ __forceinline__ void sequence(const Args& a, int b_) {
            b = b_;
            count = a.counts ? min(max(((constant_ints)a.counts)[b], 0), a.tokens) : a.tokens;
            const int total = max(((constant_ints)a.lengths)[b], 0);
            length = count ? min(total, a.c.capacity()) : 0;
            older = min(total, 1 << 30) - count;      // entry older + t is token t's own
            per_head = idx::cache4_units(length, UNIT);
        }
    };
    int before, per_head, left = end - begin;
    Unit now;
    now.sequence(a, lengths.find(begin, before, per_head));
    now.h = (begin - before) / per_head;
    now.unit = (begin - before) % per_head;
    // the keys, and where the entries' weights lie: a lane has half of an entry's elements, whole groups of 32 or one.  The next unit's are on their way
    // while one is worked on
    uint4 codes[D / 64];
    uint32_t bytes[D / 64];
    float* weight;
    const auto fetch = [&](const Unit& u) {
        const int j0 = u.unit * UNIT + wave * COLUMNS, j = j0 + r32;
        const constant_ints table = (constant_ints)(c.table + u.b * c.table_stride);
        int page = -1;
        if (j0 < u.length) {
            const int low = table[j0 >> c.log2_page], high = table[min(j0 + 16, c.capacity() - 1) >> c.log2_page];
            page = r32 < 16 ? low : high;
        }
        const bool there = j < u.length && (unsigned)page < (unsigned)c.pages;
        const int64_t block = (int64_t)(there ? page : 0) * c.heads + u.h;
        const uint8_t* const from = c.pool + block * c.block_bytes;
        const int row = j & (c.page - 1);
#pragma unroll
        for (int g = 0; g < D / 64; ++g) {
            codes[g] = *reinterpret_cast<const uint4*>(from + idx::cache4_codes(c.page, D, 0, row) + half * (D / 4) + g * 16);
            bytes[g] = from[idx::cache4_scales(c.page, D, 0, row) + half * (D / 64) + g];
            if (!there) bytes[g] = 0;
        }
        weight = there ? c.weights + block * c.page + row : nullptr;
    };
    fetch(now);
    int staged_b = -1, staged_h = -1;       // the head whose queries lie in LDS, all of them
    while (true) {
        const int b = now.b, h = now.h, length = now.length, count = now.count, rows = count * a.group, older = now.older;
        const int unit0 = now.unit * UNIT, j0 = unit0 + wave * COLUMNS, j = j0 + r32;
        v8bf k[STEPS];      // the queries' elements are taken in the same order
#pragma unroll
        for (int g = 0; g < D / 64; ++g) {
            const float scale = scale_of(bytes[g]);
            const uint32_t w[4] = {codes[g].x, codes[g].y, codes[g].z, codes[g].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 y = decode8(w[i], scale);
                k[g * 4 + i] = operand(make_uint4(y.x ^ flip, y.y ^ flip, y.z ^ flip, y.w ^ flip));
            }
        }
        float* const this_weight = weight;
        if (--left > 0) {
            if (++now.unit == now.per_head) {
                now.unit = 0;
                if (++now.h == c.heads) {
                    now.h = 0;
                    now.sequence(a, b + 1);
                }
            }
            fetch(now);
        }
        // from the first token that sees the unit's first entry, where the rows do not all fit into a tile
        const int first = rows <= ROWS ? 0 : idx::cache4_first_row(unit0, older, a.group) / 32 * 32, tiles = (rows - first + ROWS - 1) / ROWS;

        // A thread's rows are 64 apart from one tile to the next: their heads and offsets are counted on, a division each would take as long as the scores.
        // Offsets are those from the tile's first token (ti8_cache4_attention checks the strides), and none goes beyond the last row: one that is none is
        // some part of q.
        struct Place {
            int head;
            uint32_t offset;        // in bytes
        };
        int token0 = __builtin_amdgcn_readfirstlane(first / a.group), head0 = __builtin_amdgcn_readfirstlane(first % a.group);
        const auto place_of = [&](int row, int64_t st, int64_t sh) {
            return Place{(first + row) % a.group, (uint32_t)((first + row) / a.group - token0) * (uint32_t)st + (uint32_t)((first + row) % a.group) * (uint32_t)sh};
        };
        // 64 rows on, seen from a first token that is `moved` on
        const auto go_on = [&](Place& p, uint32_t st, uint32_t sh, uint32_t moved) {
            p.head += step_head;
            const bool over = p.head >= a.group;
            p.head -= over ? a.group : 0;
            p.offset += step_token * st + step_head * sh - moved * st + (over ? st - (uint32_t)a.group * sh : 0u);
        };
        const uint32_t q_st = (uint32_t)a.q_st * 2, q_sh = (uint32_t)a.q_sh * 2, lse_st = (uint32_t)a.heads * 4, lse_sh = 4;
        Place at[PASSES], at_lse = place_of(lane, lse_st, lse_sh);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = ((i * WEIGHT_WAVES + wave) * 64 + lane) / CHUNKS;
            at[i] = place_of(row, q_st, q_sh);
            at[i].offset += ((lane % CHUNKS) ^ Values<D>::swizzle(row)) * 16;
        }
        const auto issue = [&](int stage) {
            const int at_token = min(token0, count - 1), tokens = min(count - at_token, ROWS / a.group + 2);
            const auto last_of = [&](uint32_t st, uint32_t sh) { return (tokens - 1) * st + (a.group - 1) * sh; };
            const int8_t* const bq = reinterpret_cast<const int8_t*>(a.q + b * a.q_sb + at_token * a.q_st + h * a.group * a.q_sh);
            const int8_t* const bl = reinterpret_cast<const int8_t*>(a.lse + ((int64_t)b * a.tokens + at_token) * a.heads + h * a.group);
            const uint32_t rq = last_of(q_st, q_sh) + 2 * D - 16, rl = last_of(lse_st, lse_sh);
            int more = head0 + step_head >= a.group;
            head0 += step_head - (more ? a.group : 0);
            more += step_token;
            token0 += more;
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
                __builtin_amdgcn_global_load_lds(bq + min(at[i].offset, rq), queries(stage) + (i * WEIGHT_WAVES + wave) * 1024, 16, 0, 0);
            __builtin_amdgcn_global_load_lds(bl + min(at_lse.offset, rl), reinterpret_cast<int8_t*>(lses(stage)), 4, 0, 0);
            if (step_head) {        // (where a tile is whole tokens, offsets from its first stay as they are)
#pragma unroll
                for (int i = 0; i < PASSES; ++i) go_on(at[i], q_st, q_sh, more);
                go_on(at_lse, lse_st, lse_sh, more);
            }
        };

        float sum = 0.0f;
        const auto add_up = [&](int row0, int stage) {
            // somebody of these rows sees one of the wave's entries
            if (j0 >= length || row0 + ROWS <= idx::cache4_first_row(j0, older, a.group)) return;
            const int chunk = half * (D / 16) ^ Values<D>::swizzle(r32), sees = idx::cache4_first_row(j, older, a.group) - row0;        // sees: the first row that sees this lane's entry
            const auto scores = [&](int u) {
                const int8_t* const from = queries(stage) + (u * 32 + r32) * ROW;
                v16f s;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
                for (int x = 0; x < STEPS; ++x) s = mfma32(*reinterpret_cast<const v8bf*>(from + ((chunk ^ x) << 4)), k[x], s);
                return s;
            };
            const auto exponentials = [&](const v16f& s, int u, int g, auto edge) {
                const v4f shift = *reinterpret_cast<const v4f*>(lses(stage) + u * 32 + 8 * g + 4 * half);
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = u * 32 + 8 * g + 4 * half + i;
                    p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + i], factor, -shift[i]));
                    if (edge) p[i] = row >= sees && row0 + row < rows ? p[i] : 0.0f;
                }
                return (p[0] + p[1]) + (p[2] + p[3]);
            };
            if (row0 + ROWS <= rows && row0 >= idx::cache4_first_row(j0 + COLUMNS - 1, older, a.group)) {      // every row is one and sees every entry
#pragma unroll
                for (int u = 0; u < ROWS / 32; ++u) {
                    const v16f s = scores(u);
#pragma unroll
                    for (int g = 0; g < 4; ++g) sum += exponentials(s, u, g, std::false_type{});
                }
                return;
            }
#pragma unroll
            for (int u = 0; u < ROWS / 32; ++u) {
                if (row0 + u * 32 >= rows) break;
                const v16f s = scores(u);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (row0 + u * 32 + 8 * g >= rows) break;       // (a step's few rows: no exponentials of rows that are none)
                    sum += exponentials(s, u, g, std::true_type{});
                }
            }
        };
        if (rows <= ROWS) {
            if (rows > 0 && (b != staged_b || h != staged_h)) {
                wait_and_meet<0>();
                issue(0);
                wait_and_meet<0>();
                lses(0)[lane] *= LOG2E;
                staged_b = b;
                staged_h = h;
            }
            if (rows > 0) add_up(0, 0);
        } else {
            staged_b = -1;
            wait_and_meet<0>();     // from here on nothing but the tiles' loads is in flight: the loop counts them
            issue(0);
            issue(1);
            for (int t = 0, stage = 0; t < tiles; ++t) {
                wait_and_meet<LOADS>();       // tile t is there, and nobody reads tile t - 1, whose place is the next one's
                issue(stage == 0 ? RING - 1 : stage - 1);
                lses(stage)[lane] *= LOG2E;
                add_up(first + t * ROWS, stage);
                stage = stage == RING - 1 ? 0 : stage + 1;
            }
            __builtin_amdgcn_s_waitcnt(0);      // the loads behind the last tile: LDS may be another workgroup's once the wave has ended
        }
        sum = over_halves<true>(sum);
        if (this_weight && half == 0) unsafeAtomicAdd(this_weight, sum);       // (device memory: global_atomic_add_f32)
        if (left <= 0) break;
    }
#endif
}

// Workgroups of step_kernel: as many as run at a time (three per CU with 16 rows, two with 32: their registers), and no more than there are units
int step_groups(const Cache& c, int tiles) {
    const int64_t units = (int64_t)c.batch * c.heads * (idx::cache4_units(c.capacity(), idx::CACHE4_UNIT) + EXTRA), most = device_cu_count() * (tiles == 1 ? 3 : 2);
    return (int)(units < most ? units : most);
}
// Whether every (sequence, head) is left to a workgroup of its own, which saves the join and the search for its entries, but nobody helps with a long
// sequence (us, shared out / each its own; heads of 128, one token).  8 heads of 512 entries 10.6 / 7.8, of 1024 10.5 / 10.3, of 2048 10.8 / 16.7; 256 heads
// of 1024 18.0 / 12.3, of 2048 23.6 / 19.6 (of 1 to 2048 17.5 / 18.0), of 2560 26.5 / 22.5 (of 1 to 2560 19.4 / 21.5), of 4096 34.6 / 31.9 (of 1 to 4096 19.4 / 30.5); 192 heads of 2560
// 22.7 / 21.6, of 4096 28.6 / 31.0; 128 heads of 2048 17.8 / 17.8, of 2560 18.7 / 21.0.  So 2048 is where sequences of several lengths, and 128 heads, take as long either
// way; the host sees the room alone, and full sequences of 256 heads beyond it would lose less than those of several lengths gain.  In two rounds, 512 heads of
// 256 entries 15.1 / 11.2, of 512 18.0 / 16.1, of 1024 23.6 / 22.4 (of 1 to 1024 19.2 / 20.2)
bool step_alone(const Cache& c, int tiles) {
    const int64_t pairs = (int64_t)c.batch * c.heads, room = device_cu_count() * (c.dim == 64 && tiles == 1 ? 2 : 1);      // (registers)
    return pairs <= room ? c.capacity() <= (3 * pairs > 2 * room ? 2048 : 1024) : pairs <= 2 * room && c.capacity() <= 512;
}
// Row tiles of step_kernel that hold all rows of a kv head (1 or 2), or 0: prompt_kernel.  Four of them take longer than it, 4 streams of 16384 entries and
// 64 rows 62 us to 54; two less, 16 streams of 8192 and 32 rows 57 to 76
int step_tiles(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 0; }

// prompt_kernel: waves of a workgroup, how many of them have the same rows, and how many workgroups share the entries of a row block.  Heads of 128: eight waves
// convert every entry for 256 rows and have a CU to themselves; four, two workgroups of which a CU holds, are taken where the eight would hold 128 more rows that
// are none (us with four / eight waves, 32 heads: 9 x 600 rows over 2000 entries 211 / 246, 3 x 600 112 / 116, 6 x 1150 214 / 222, 40 x 280 of 8 heads 152 / 190, the worst of
// 14 sizes 6 x 890 187 / 180; where none are saved, 8 x 512 rows of 8 heads over 4096 entries 173 / 160, 2 x 8192 of 8 heads 493 / 466, 3 x 1024 117 / 117).  Heads
// of 64: four waves, whose registers a CU holds three times (1000 tokens over 2000 entries 45 -> 40 us).
// Up to 64 rows two and two of the four share the rows (4 streams of 16384 entries, 64 rows: 49 -> 45 us).  Parts are worth it from 4 tiles of entries on.
struct PromptPlan {
    int waves, shares, blocks, splits, shared_from;
};
PromptPlan prompt_plan(const Cache& c, int64_t rows) {
    const int64_t pairs = (int64_t)c.batch * c.heads, cus = device_cu_count();
    PromptPlan p;
    p.waves = c.dim == 128 && (rows + 127) / 128 % 2 == 0 ? 8 : 4;
    p.shares = rows <= 64 ? 2 : 1;
    p.blocks = (int)((rows * p.shares + p.waves * 32 - 1) / (p.waves * 32));
    const int64_t groups = pairs * p.blocks, room = cus * (c.dim == 64 ? 3 : 8 / p.waves), most = (c.capacity() + 4 * TILE - 1) / (4 * TILE);
    // One part, or as many as fill the CUs once, twice or three times, by an estimate in us: 2 per tile of entries in a row, parts written and read at two thirds
    // of the rate of a copy (12 x 280 rows of 8 heads over 4000 entries 134 -> 117 us in three parts, 24 x 64 of 1 to 4000 55 -> 50 in two).  Sequences may be far shorter than their
    // tables: the kernel leaves a block whole up to half of what two parts, or as many as it takes where two are no gain, need to be worth it (half: lengths differ,
    // and the longest decides; 64 rows of 8 heads, the first 64 entries of 8192: 27 -> 14 us).
    const double tiles = (double)c.capacity() / TILE, join = (double)(pairs * rows) * (c.dim + 4) * 8e-6 / 3.3;
    const auto rounds_of = [&](int64_t splits) { return (double)((groups * splits + room - 1) / room) / (double)splits; };
    double best = rounds_of(1) * tiles * 2.0;
    p.splits = 1;
    p.shared_from = 1;
    for (int rounds = 1; rounds <= 3; ++rounds) {
        const int64_t fill = rounds * room / groups, splits = fill < most ? fill : most;
        if (splits < 2 || rounds_of(splits) * tiles * 2.0 + 3.0 + join * (double)splits >= best) continue;
        best = rounds_of(splits) * tiles * 2.0 + 3.0 + join * (double)splits;
        p.splits = (int)splits;
        const int64_t fewest = 2 * groups <= room ? 2 : splits;
        p.shared_from = std::max(5, (int)((3.0 + join * (double)fewest) / (4.0 * (rounds_of(1) - rounds_of(fewest)))));
    }
    return p;
}
int64_t owners_bytes(const Cache& c) { return ((int64_t)c.batch * c.heads * (int64_t)sizeof(int2) + 15) / 16 * 16; }
int64_t workspace_bytes_of(const Cache& c, int64_t tokens, int64_t heads) {
    const int64_t rows = tokens * (heads / c.heads);
    const int tiles = step_tiles(rows);
    if (tiles && step_alone(c, tiles)) return 0;
    if (tiles) return owners_bytes(c) + (int64_t)step_groups(c, tiles) * 2 * tiles * 16 * (c.dim + 4) * (int64_t)sizeof(float);
    const PromptPlan p = prompt_plan(c, rows);
    return p.splits > 1 ? c.batch * tokens * heads * p.splits * (c.dim + 4) * (int64_t)sizeof(float) : 0;
}

template <int D, int TILES>
int launch_step(const char* fn, Args& a, hipStream_t st) {
    if (step_alone(a.c, TILES)) {
        hipLaunchKernelGGL((step_kernel<D, TILES, true>), dim3((unsigned)(a.c.batch * a.c.heads)), dim3(2 * WAVES * 64), 0, st, a);
        return check_launch(fn);
    }
    a.groups = step_groups(a.c, TILES);
    a.owners = reinterpret_cast<int2*>(a.parts);
    a.parts += owners_bytes(a.c) / (int64_t)sizeof(float);
    hipLaunchKernelGGL((step_kernel<D, TILES, false>), dim3((unsigned)a.groups), dim3(WAVES * 64), 0, st, a);
    if (int e = check_launch(fn)) return e;
    hipLaunchKernelGGL((join_kernel<D, TILES>), dim3((unsigned)(a.c.batch * a.c.heads * a.tokens * a.group)), dim3(256), 0, st, a);
    return check_launch(fn);
}

template <int D, int NW, int SHARES>
int prepare_prompt(const char* fn) {
    static OncePerDevice once;
    const hipError_t e = raise_lds_limit(once, reinterpret_cast<const void*>(prompt_kernel<D, NW, SHARES>), PROMPT_STAGES<NW> * 2 * Tile32<D>::BYTES);
    return e == hipSuccess ? TI8_OK : fail(TI8_ERR_HIP, "%s: cannot raise the LDS limit: %s", fn, hipGetErrorString(e));
}

template <int D, int NW, int SHARES>
int launch_prompt(const char* fn, const Args& a, hipStream_t st) {
    if (int e = prepare_prompt<D, NW, SHARES>(fn)) return e;
    const int64_t grid = idx::round8((int64_t)a.c.batch * a.c.heads) * a.blocks * a.splits;
    hipLaunchKernelGGL((prompt_kernel<D, NW, SHARES>), dim3((unsigned)grid), dim3(NW * 64), PROMPT_STAGES<NW> * 2 * Tile32<D>::BYTES, st, a);
    if (int e = check_launch(fn)) return e;
    if (a.splits == 1) return TI8_OK;
    // a whole workgroup for a row of many parts (64 of them: 3 us; 30 where their loads follow each other)
    const int64_t rows = (int64_t)a.c.batch * a.tokens * a.heads, per = 1024 / D;
    if (a.splits > 8) hipLaunchKernelGGL((join_rows_kernel<D, 1024 / D>), dim3((unsigned)rows), dim3(256), 0, st, a, rows);
    else hipLaunchKernelGGL((join_rows_kernel<D, 1>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, st, a, rows);
    return check_launch(fn);
}

template <int D>
int launch(const char* fn, Args& a, bool accumulate, hipStream_t st) {
    const int64_t rows = (int64_t)a.tokens * a.group;
    const int tiles = step_tiles(rows);
    int e;
    if (tiles) {
        e = tiles == 1 ? launch_step<D, 1>(fn, a, st) : launch_step<D, 2>(fn, a, st);
    } else {
        const PromptPlan p = prompt_plan(a.c, rows);
        a.blocks = p.blocks;
        a.block_rows = p.waves / p.shares * 32;
        a.splits = p.splits;
        a.shared_from = p.shared_from;
        if (p.shares == 2) e = launch_prompt<D, 4, 2>(fn, a, st);
        else if (D == 128 && p.waves == 8) e = launch_prompt<128, 8, 1>(fn, a, st);
        else e = launch_prompt<D, 4, 1>(fn, a, st);
    }
    if (e || !accumulate) return e;
    const int64_t units = (int64_t)a.c.batch * a.c.heads * idx::cache4_units(a.c.capacity(), WEIGHTS_UNIT), most = device_cu_count() * 2;
    a.groups = (int)(units < most ? units : most);
    hipLaunchKernelGGL((weights_kernel<D>), dim3((unsigned)a.groups), dim3(WEIGHT_WAVES * 64), 0, st, a);
    return check_launch(fn);
}

}  // namespace

int init_attention() {
    const char* fn = "ti8_init";
    int e = prepare_prompt<128, 8, 1>(fn);
    if (!e) e = prepare_prompt<128, 4, 1>(fn);
    if (!e) e = prepare_prompt<128, 4, 2>(fn);
    if (!e) e = prepare_prompt<64, 4, 1>(fn);
    return e ? e : prepare_prompt<64, 4, 2>(fn);
}

}  // namespace cache4
}  // namespace ti8

using namespace ti8;
using namespace ti8::cache4;

extern "C" int64_t ti8_cache4_attention_workspace(const ti8_cache4* p, int64_t tokens, int64_t heads) {
    Cache c;
    if (check("ti8_cache4_attention_workspace", p, c)) return -1;
    if (tokens <= 0 || tokens > (1 << 24) || heads <= 0 || heads % c.heads || heads / c.heads > 4096 || c.batch * tokens * heads > 0x3fffffff ||
        (int64_t)c.batch * c.heads * (idx::cache4_units(c.capacity(), idx::CACHE4_UNIT) + EXTRA) > 0x3fffffff)
        return -1;
    if (idx::round8((int64_t)c.batch * c.heads) * ((tokens * (heads / c.heads) + 127) / 128) > 0x3fffffff) return -1;
    return workspace_bytes_of(c, tokens, heads);
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
    if (!(scale >= -0x1p127f && scale <= 0x1p127f)) return fail(TI8_ERR_SHAPE, "%s: scale must be a number of up to 2^127 in magnitude, got %g", fn, (double)scale);
    if (!q || !lengths || !out || !lse || (accumulate && !c.weights) || (need && !workspace))
        return fail(TI8_ERR_NULL, "%s: q, lengths, out and lse are required, the weights to add up as well, and the workspace", fn);
    if (need > workspace_bytes) return fail(TI8_ERR_SHAPE, "%s: %lld bytes of workspace are needed, got %lld", fn, (long long)need, (long long)workspace_bytes);
    if (!aligned16(q) || !aligned16(out) || (reinterpret_cast<uintptr_t>(lse) & 3) || !aligned16(workspace) || q_stride_b % 8 || q_stride_t % 8 || q_stride_h % 8)
        return fail(TI8_ERR_ALIGN, "%s: q, out and the workspace must be 16-byte aligned, q's strides multiples of 8 elements", fn);
    // weights_kernel: 32-bit offsets within a tile's rows
    const int64_t group = heads / c.heads, tile_tokens = ROWS / group + 2;
    const auto within = [&](int64_t st, int64_t sh) { return st >= 0 && sh >= 0 && st <= 0x3fffffff / tile_tokens && sh <= 0x3fffffff / group && tile_tokens * st + group * sh + c.dim <= 0x3fffffff; };
    if (accumulate && (!within(q_stride_t, q_stride_h) || !within(heads, 1)))
        return fail(TI8_ERR_SHAPE, "%s: q's strides of %lld and %lld elements between tokens and heads are too large for the weights to be added up", fn,
                    (long long)q_stride_t, (long long)q_stride_h);
    Args a{c, lengths, counts, static_cast<const uint16_t*>(q), q_stride_b, q_stride_t, q_stride_h, static_cast<uint16_t*>(out), lse, nullptr, static_cast<float*>(workspace),
           (int)tokens, (int)heads, (int)(heads / c.heads), scale, 0, 0, 0};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return c.dim == 128 ? launch<128>(fn, a, accumulate != 0, st) : launch<64>(fn, a, accumulate != 0, st);
}
