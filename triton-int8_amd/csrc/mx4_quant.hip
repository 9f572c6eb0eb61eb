// Quantisers into 4 bits with shared scales (format: mx4.h), the values back, and the norm whose result is quantised on the way out.  All are bound by HBM:
// every input is read once and every output written once.
#include "mx4.h"
#include "quant_math.h"

namespace ti8 {
namespace mx4 {
namespace {

constexpr int THREADS = 256;

struct QuantArgs {
    const uint16_t* x;
    int64_t ldx, R, C;
    Tensor rows, cols;
};

// By rows: 32 rows x 256 columns per workgroup; a row's 512 bytes are read by half a wave, a group's maximum is over four lanes.
__global__ __launch_bounds__(THREADS) void quant_row_kernel(QuantArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t tiles = idx::mx4_tiles(g.C), tile = blockIdx.x % tiles, row0 = (int64_t)(blockIdx.x / tiles) * idx::MX4_ROW_BLOCK + (threadIdx.x >> 5);
    const int octet = threadIdx.x & 31;
    const int64_t col = tile * idx::MX4_TILE + octet * 8;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = row0 + 8 * i < g.R ? load8(g.x + (row0 + 8 * i) * g.ldx + col, g.C - col) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + 8 * i;
        const uint32_t byte = scale_byte(quad_max(halves_max(largest2(v[i]))));
        if (row >= g.R) continue;
        *reinterpret_cast<uint32_t*>(g.rows.codes + idx::mx4_code_at(row, g.rows.ld, tile, octet)) = encode8(v[i].x, v[i].y, v[i].z, v[i].w, byte);
        if ((octet & 3) == 0) g.rows.scales[idx::mx4_scale_at(tile, g.rows.scale_ld, row, octet >> 2)] = (uint8_t)byte;
    }
#else
    (void)g;
#endif
}

// By columns (the transposed tensor's rows), with ROWS both ways from the same read: 32 rows x 256 columns per wave, a lane has 8 columns of 16 rows in
// registers.  A column's group is two lanes' (l and l + 32); its codes go through LDS, from where lines of a column are written.
template <int NW, bool ROWS>
__global__ __launch_bounds__(64 * NW) void quant_cols_kernel(QuantArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int LINE = NW * 16;                       // bytes of a column's codes here
    __shared__ __attribute__((aligned(16))) uint8_t lines[idx::MX4_TILE * LINE];
    __shared__ __attribute__((aligned(16))) uint8_t row_scales[32 * NW * 8], col_scales[idx::MX4_TILE * NW];
    const int64_t tiles = idx::mx4_tiles(g.C), tile = blockIdx.x % tiles, chunk = blockIdx.x / tiles;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, octet = lane & 31, half = lane >> 5;
    const int64_t col = tile * idx::MX4_TILE + octet * 8, first = chunk * (32 * NW), row0 = first + wave * 32 + half * 16;
    uint4 v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = row0 + i < g.R ? load8(g.x + (row0 + i) * g.ldx + col, g.C - col) : make_uint4(0, 0, 0, 0);
    if (ROWS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t byte = scale_byte(quad_max(halves_max(largest2(v[i]))));
            if (row0 + i < g.R)
                *reinterpret_cast<uint32_t*>(g.rows.codes + idx::mx4_code_at(row0 + i, g.rows.ld, tile, octet)) = encode8(v[i].x, v[i].y, v[i].z, v[i].w, byte);
            if ((octet & 3) == 0) row_scales[(wave * 32 + half * 16 + i) * 8 + (octet >> 2)] = (uint8_t)byte;
        }
    }
    uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        m[0] = pk_max(m[0], v[i].x & MAGNITUDE);
        m[1] = pk_max(m[1], v[i].y & MAGNITUDE);
        m[2] = pk_max(m[2], v[i].z & MAGNITUDE);
        m[3] = pk_max(m[3], v[i].w & MAGNITUDE);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = pk_max(m[j], (uint32_t)__shfl_xor((int)m[j], 32, 64));
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const uint32_t byte = scale_byte(odd ? m[j] >> 16 : m[j] & 0xffffu);
            const auto pair = [&](int i) {      // rows i and i + 1 of this column
                const uint32_t a = j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w, b = j == 0 ? v[i + 1].x : j == 1 ? v[i + 1].y : j == 2 ? v[i + 1].z : v[i + 1].w;
                return odd ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
            };
            const uint2 w = make_uint2(encode8(pair(0), pair(2), pair(4), pair(6), byte), encode8(pair(8), pair(10), pair(12), pair(14), byte));
            const int c = octet * 8 + 2 * j + odd;
            *reinterpret_cast<uint2*>(lines + c * LINE + idx::mx4_col_chunk(wave, octet, NW) * 16 + half * 8) = w;
            if (half == 0) col_scales[c * NW + wave] = (uint8_t)byte;
        }
    }
    __syncthreads();
    if (ROWS) {
        const int64_t row = first + threadIdx.x;
        if (threadIdx.x < 32 * NW && row < g.R)
            *reinterpret_cast<uint2*>(g.rows.scales + idx::mx4_scale_at(tile, g.rows.scale_ld, row, 0)) = *reinterpret_cast<const uint2*>(row_scales + threadIdx.x * 8);
    }
    const int64_t row_tile = first / idx::MX4_TILE;
    const int within = (int)(first % idx::MX4_TILE) / 2, group = (int)(first % idx::MX4_TILE) / 32;
#pragma unroll
    for (int u = 0; u < 4; ++u) {       // 256 columns of NW pieces of 16 bytes
        const int piece = u * 64 * NW + threadIdx.x, c = piece / NW, p = piece % NW;
        const int64_t at = tile * idx::MX4_TILE + c;
        if (at < g.C)
            *reinterpret_cast<uint4*>(g.cols.codes + at * g.cols.ld + row_tile * idx::MX4_TILE_BYTES + within + p * 16) =
                *reinterpret_cast<const uint4*>(lines + c * LINE + idx::mx4_col_chunk(p, c >> 3, NW) * 16);
    }
    for (int c = threadIdx.x; c < idx::MX4_TILE; c += 64 * NW) {
        const int64_t at = tile * idx::MX4_TILE + c;
        if (at >= g.C) break;
        uint8_t* to = g.cols.scales + idx::mx4_scale_at(row_tile, g.cols.scale_ld, at, group);
        if (NW == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(col_scales + c * NW);
        else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(col_scales + c * NW);
    }
#else
    (void)g;
#endif
}

// The values back, exact in bf16
__global__ __launch_bounds__(THREADS) void dequant_kernel(Tensor q, int64_t R, int64_t C, uint16_t* __restrict__ y, int64_t ldy) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t tiles = idx::mx4_tiles(C), tile = blockIdx.x % tiles, row0 = (int64_t)(blockIdx.x / tiles) * idx::MX4_ROW_BLOCK + (threadIdx.x >> 5);
    const int octet = threadIdx.x & 31;
    const int64_t col = tile * idx::MX4_TILE + octet * 8;
    if (col >= C) return;
    uint32_t w[4], byte[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + 8 * i;
        w[i] = byte[i] = 0;
        if (row < R) {
            w[i] = *reinterpret_cast<const uint32_t*>(q.codes + idx::mx4_code_at(row, q.ld, tile, octet));
            byte[i] = q.scales[idx::mx4_scale_at(tile, q.scale_ld, row, octet >> 2)];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + 8 * i;
        if (row >= R) break;
        const float scale = scale_of(byte[i]);
        uint4 v;
        v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale, 0));
        v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale, 1));
        v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale, 2));
        v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[i], scale, 3));
        if (byte[i] == NAN_SCALE) v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        store8(y + row * ldy + col, v, C - col);
    }
#else
    (void)q; (void)R; (void)C; (void)y; (void)ldy;
#endif
}

// int8 codes with a scale per row (group 0) or per 128 columns back to bf16, eight elements per thread
__global__ __launch_bounds__(THREADS) void dequant_row_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ s, int64_t rows, int64_t cols, int by_group,
                                                              uint16_t* __restrict__ y, int64_t ldy) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t octets = cols >> 3, at = (int64_t)blockIdx.x * THREADS + threadIdx.x, row = at / octets, o = at - row * octets;
    if (row >= rows) return;
    const uint2 w = *reinterpret_cast<const uint2*>(q + row * ldq + o * 8);
    const float scale = by_group ? s[row * (cols >> 7) + (o >> 4)] : s[row];
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * scale;
    *reinterpret_cast<uint4*>(y + row * ldy + o * 8) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
#else
    (void)q; (void)ldq; (void)s; (void)rows; (void)cols; (void)by_group; (void)y; (void)ldy;
#endif
}

enum { TO_MX4 = 0, TO_ROW = 1, TO_GROUP = 2 };

struct NormArgs {
    const uint16_t *x, *residual, *w;
    int64_t ldx, ldr, ldh, rows;
    uint16_t* h;
    float* rstd;
    int dim;
    double eps;
    Tensor mx;
    int8_t* q;
    int64_t ldq;
    float* s;
    QMode mode;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
}

// h = bf16(x + residual), r = 1 / sqrt(mean(h^2) + eps), y = bf16(bf16(h r) w), quantised: a row in the registers of T threads (64: four rows to a workgroup),
// NV octets each.  The squares are added up in 64 bits (they are exact in it) and r is rounded to 32 once: no code depends on an order of summation.
template <int T, int NV, int TO>
__global__ __launch_bounds__(THREADS) void rmsnorm_quant_kernel(NormArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ double sums[4];
    __shared__ float red[4];
    const int64_t row = idx::xcd_range(blockIdx.x, gridDim.x) * (THREADS / T) + threadIdx.x / T;
    if (row >= g.rows) return;          // (whole waves; the whole workgroup where it shares a row)
    const int t = threadIdx.x % T, octets = g.dim >> 3;
    uint4 v[NV];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int o = t + i * T;
        v[i] = make_uint4(0, 0, 0, 0);
        if (o < octets) {
            v[i] = load16(g.x + row * g.ldx + o * 8);
            if (g.residual) {
                const uint4 b = load16(g.residual + row * g.ldr + o * 8);
                v[i] = make_uint4(add_bf16x2(v[i].x, b.x), add_bf16x2(v[i].y, b.y), add_bf16x2(v[i].z, b.z), add_bf16x2(v[i].w, b.w));
                *reinterpret_cast<uint4*>(g.h + row * g.ldh + o * 8) = v[i];
            }
        }
    }
    const auto word = [&](int i, int j) { return j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w; };
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = bf16_lo(word(i, j)), b = bf16_hi(word(i, j));
            sum = __builtin_fma(a, a, sum);
            sum = __builtin_fma(b, b, sum);
        }
    sum = wave_sum(sum);
    if (T > 64) {
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
        __syncthreads();
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    const float r = (float)(1.0 / sqrt(sum / (double)g.dim + g.eps));
    if (t == 0) g.rstd[row] = r;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int o = t + i * T;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (o < octets) w = load16(g.w + o * 8);
        const auto scaled = [&](uint32_t h2, uint32_t w2) {
            const uint32_t n = pack_bf16x2(bf16_lo(h2) * r, bf16_hi(h2) * r);
            return pack_bf16x2(bf16_lo(n) * bf16_lo(w2), bf16_hi(n) * bf16_hi(w2));
        };
        v[i] = o < octets ? make_uint4(scaled(v[i].x, w.x), scaled(v[i].y, w.y), scaled(v[i].z, w.z), scaled(v[i].w, w.w)) : make_uint4(0, 0, 0, 0);
        if (TO == TO_MX4) {
            const uint32_t byte = scale_byte(quad_max(halves_max(largest2(v[i]))));
            if (o < (int)idx::mx4_tiles(g.dim) * 32) {
                *reinterpret_cast<uint32_t*>(g.mx.codes + idx::mx4_code_at(row, g.mx.ld, o >> 5, o & 31)) = encode8(v[i].x, v[i].y, v[i].z, v[i].w, byte);
                if ((o & 3) == 0) g.mx.scales[idx::mx4_scale_at(o >> 5, g.mx.scale_ld, row, (o & 31) >> 2)] = (uint8_t)byte;
            }
        } else if (TO == TO_GROUP) {
            const float floored = amax_floor(row16_max(absmax8(v[i], 0.0f)), g.mode.eps_add), scale = 127.0f / floored;
            if (o < octets) {
                *reinterpret_cast<uint2*>(g.q + row * g.ldq + o * 8) = quant8(v[i], scale);
                if ((o & 15) == 0) g.s[row * (g.dim >> 7) + (o >> 4)] = stored_scale(floored, scale, g.mode);
            }
        } else {
            amax = absmax8(v[i], amax);
        }
    }
    if (TO == TO_ROW) {
        amax = T > 64 ? block_max_256(amax, red) : wave_max(amax);
        const float floored = amax_floor(amax, g.mode.eps_add), scale = 127.0f / floored;
        if (t == 0) g.s[row] = stored_scale(floored, scale, g.mode);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int o = t + i * T;
            if (o < octets) *reinterpret_cast<uint2*>(g.q + row * g.ldq + o * 8) = quant8(v[i], scale);
        }
    }
#else
    (void)g;
#endif
}

constexpr int NORM_MAX_DIM = THREADS * 8 * 8;

template <int TO>
void launch_norm(const NormArgs& g, hipStream_t st) {
    const auto go = [&](auto kernel, int rows_per_group) { kernel<<<dim3((unsigned)((g.rows + rows_per_group - 1) / rows_per_group)), dim3(THREADS), 0, st>>>(g); };
    if (g.dim <= 512) go(rmsnorm_quant_kernel<64, 1, TO>, 4);
    else if (g.dim <= 1024) go(rmsnorm_quant_kernel<64, 2, TO>, 4);
    else if (g.dim <= 2048) go(rmsnorm_quant_kernel<THREADS, 1, TO>, 1);
    else if (g.dim <= 4096) go(rmsnorm_quant_kernel<THREADS, 2, TO>, 1);
    else if (g.dim <= 8192) go(rmsnorm_quant_kernel<THREADS, 4, TO>, 1);
    else go(rmsnorm_quant_kernel<THREADS, 8, TO>, 1);
}

bool grid_ok(int64_t blocks) { return blocks > 0 && blocks <= 0x7fffffff; }

}  // namespace
}  // namespace mx4
}  // namespace ti8

using namespace ti8;

extern "C" int ti8_mx4_quant(const void* x, int64_t ldx, int64_t rows, int64_t cols, const ti8_mx4* by_rows, const ti8_mx4* by_columns, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_quant";
    if (!x || (!by_rows && !by_columns)) return fail(TI8_ERR_NULL, "%s: x and one of by_rows and by_columns are required", fn);
    if (rows <= 0 || cols <= 0 || rows > (1 << 28) || cols > (1 << 28) || (rows > 1 && ldx < cols))
        return fail(TI8_ERR_SHAPE, "%s: need rows, cols in 1 .. 2^28 and ldx >= cols; got rows=%lld cols=%lld ldx=%lld", fn, (long long)rows, (long long)cols, (long long)ldx);
    if (reinterpret_cast<uintptr_t>(x) & 1) return fail(TI8_ERR_ALIGN, "%s: x must be 2-byte aligned", fn);
    mx4::QuantArgs g{static_cast<const uint16_t*>(x), ldx, rows, cols, {}, {}};
    if (by_rows)
        if (int e = mx4::check(fn, "by_rows", by_rows, rows, cols, g.rows)) return e;
    if (by_columns)
        if (int e = mx4::check(fn, "by_columns", by_columns, cols, rows, g.cols)) return e;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t tiles = idx::mx4_tiles(cols);
    if (!by_columns) {
        const int64_t blocks = tiles * ((rows + idx::MX4_ROW_BLOCK - 1) / idx::MX4_ROW_BLOCK);
        if (!mx4::grid_ok(blocks)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
        mx4::quant_row_kernel<<<dim3((unsigned)blocks), dim3(mx4::THREADS), 0, st>>>(g);
        return check_launch(fn);
    }
    // a workgroup per 256 x 256 elements, per 64 x 256 where that would leave CUs without one
    const int64_t large = tiles * idx::mx4_tiles(rows);
    const bool small = large < 2 * device_cu_count();
    const int64_t blocks = small ? 4 * large : large;
    if (!mx4::grid_ok(blocks)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    const auto go = [&](auto kernel, int waves) { kernel<<<dim3((unsigned)blocks), dim3(64 * waves), 0, st>>>(g); };
    if (small) by_rows ? go(mx4::quant_cols_kernel<2, true>, 2) : go(mx4::quant_cols_kernel<2, false>, 2);
    else by_rows ? go(mx4::quant_cols_kernel<8, true>, 8) : go(mx4::quant_cols_kernel<8, false>, 8);
    return check_launch(fn);
}

extern "C" int ti8_mx4_dequant(const ti8_mx4* q, int64_t rows, int64_t cols, void* y, int64_t ldy, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_dequant";
    if (!q || !y) return fail(TI8_ERR_NULL, "%s: q and y are required", fn);
    if (rows <= 0 || cols <= 0 || rows > (1 << 28) || cols > (1 << 28) || (rows > 1 && ldy < cols))
        return fail(TI8_ERR_SHAPE, "%s: need rows, cols in 1 .. 2^28 and ldy >= cols; got rows=%lld cols=%lld ldy=%lld", fn, (long long)rows, (long long)cols, (long long)ldy);
    if (reinterpret_cast<uintptr_t>(y) & 1) return fail(TI8_ERR_ALIGN, "%s: y must be 2-byte aligned", fn);
    mx4::Tensor t;
    if (int e = mx4::check(fn, "q", q, rows, cols, t)) return e;
    const int64_t blocks = idx::mx4_tiles(cols) * ((rows + idx::MX4_ROW_BLOCK - 1) / idx::MX4_ROW_BLOCK);
    if (!mx4::grid_ok(blocks)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    mx4::dequant_kernel<<<dim3((unsigned)blocks), dim3(mx4::THREADS), 0, static_cast<hipStream_t>(stream)>>>(t, rows, cols, static_cast<uint16_t*>(y), ldy);
    return check_launch(fn);
}

extern "C" int ti8_dequant_row(const int8_t* q, int64_t ldq, const float* s, int64_t rows, int64_t cols, int group, void* y, int64_t ldy, ti8_stream_t stream) {
    const char* const fn = "ti8_dequant_row";
    if (!q || !s || !y) return fail(TI8_ERR_NULL, "%s: q, s and y are required", fn);
    if (rows <= 0 || cols <= 0 || rows > (1 << 28) || cols > (1 << 28) || cols % 8 || (group && cols % 128) || ldq < cols || ldy < cols)
        return fail(TI8_ERR_SHAPE, "%s: need rows, cols in 1 .. 2^28, cols%%8==0 (with groups cols%%128==0) and leading dimensions of at least cols; got rows=%lld cols=%lld ldq=%lld ldy=%lld",
                    fn, (long long)rows, (long long)cols, (long long)ldq, (long long)ldy);
    if (group != 0 && group != 128) return fail(TI8_ERR_MODE, "%s: group must be 0 or 128, got %d", fn, group);
    if ((reinterpret_cast<uintptr_t>(q) & 7) || ldq % 8 || !aligned16(y) || ldy % 8 || (reinterpret_cast<uintptr_t>(s) & 3))
        return fail(TI8_ERR_ALIGN, "%s: rows of q must be 8-byte aligned, those of y 16-byte, s 4-byte", fn);
    const int64_t blocks = (rows * (cols >> 3) + mx4::THREADS - 1) / mx4::THREADS;
    if (!mx4::grid_ok(blocks)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    mx4::dequant_row_kernel<<<dim3((unsigned)blocks), dim3(mx4::THREADS), 0, static_cast<hipStream_t>(stream)>>>(q, ldq, s, rows, cols, group ? 1 : 0, static_cast<uint16_t*>(y), ldy);
    return check_launch(fn);
}

extern "C" int ti8_rmsnorm_quant(const ti8_rmsnorm_quant_args* a, ti8_stream_t stream) {
    const char* const fn = "ti8_rmsnorm_quant";
    if (!a || !a->x || !a->w || !a->rstd) return fail(TI8_ERR_NULL, "%s: x, w and rstd are required", fn);
    if (!a->residual != !a->h) return fail(TI8_ERR_NULL, "%s: residual and h go together", fn);
    if (!a->mx4.codes == !a->q) return fail(TI8_ERR_NULL, "%s: one of mx4 and q is required", fn);
    const int64_t rows = a->rows, dim = a->dim;
    if (rows <= 0 || rows > (1 << 28) || dim <= 0 || dim % 8 || dim > mx4::NORM_MAX_DIM || a->ldx < dim || (a->residual && (a->ldr < dim || a->ldh < dim)))
        return fail(TI8_ERR_SHAPE, "%s: need rows in 1 .. 2^28, dim a multiple of 8 up to %d and leading dimensions of at least dim; got rows=%lld dim=%lld", fn, mx4::NORM_MAX_DIM,
                    (long long)rows, (long long)dim);
    if (!aligned16(a->x) || !aligned16(a->w) || !aligned16(a->residual) || !aligned16(a->h) || a->ldx % 8 || (a->residual && (a->ldr % 8 || a->ldh % 8)) ||
        (reinterpret_cast<uintptr_t>(a->rstd) & 3))
        return fail(TI8_ERR_ALIGN, "%s: rows of x, residual and h and the weight must be 16-byte aligned", fn);
    mx4::NormArgs g{static_cast<const uint16_t*>(a->x), static_cast<const uint16_t*>(a->residual), static_cast<const uint16_t*>(a->w), a->ldx, a->ldr, a->ldh, rows,
                    static_cast<uint16_t*>(a->h), a->rstd, (int)dim, a->eps, {}, a->q, a->ldq, a->s, {}};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->mx4.codes) {
        if (int e = mx4::check(fn, "mx4", &a->mx4, rows, dim, g.mx)) return e;
        mx4::launch_norm<mx4::TO_MX4>(g, st);
        return check_launch(fn);
    }
    if (!a->s) return fail(TI8_ERR_NULL, "%s: q needs s", fn);
    if (a->group != 0 && a->group != 128) return fail(TI8_ERR_MODE, "%s: group must be 0 or 128, got %d", fn, a->group);
    if (a->qflags & ~(TI8_Q_CLAMP | TI8_Q_EPS_ADD | TI8_Q_SCALE_BF16)) return fail(TI8_ERR_MODE, "%s: quantiser flags 0x%x do not apply here", fn, a->qflags);
    if (int e = parse_mode(a->qflags, a->inv_mode, &g.mode)) return e;
    if (dim % 128 || a->ldq < dim) return fail(TI8_ERR_SHAPE, "%s: int8 codes need dim%%128==0 and ldq >= dim, got dim=%lld ldq=%lld", fn, (long long)dim, (long long)a->ldq);
    if ((reinterpret_cast<uintptr_t>(a->q) & 7) || a->ldq % 8 || (reinterpret_cast<uintptr_t>(a->s) & 3)) return fail(TI8_ERR_ALIGN, "%s: rows of q must be 8-byte aligned, s 4-byte", fn);
    if (a->group) mx4::launch_norm<mx4::TO_GROUP>(g, st);
    else mx4::launch_norm<mx4::TO_ROW>(g, st);
    return check_launch(fn);
}
