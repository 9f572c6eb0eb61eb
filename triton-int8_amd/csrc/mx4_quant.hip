// Quantisers into 4 bits with shared scales (format: mx4.h), the values back, and the norm whose result is quantised on the way out.  All are bound by HBM:
// every input is read once and every output written once.
#include "mx4.h"
#include "quant_math.h"

namespace ti8 {
namespace mx4 {
namespace {

constexpr int THREADS = 256;

struct QuantOperand {
    const uint16_t* x;
    int64_t ldx, R, C;
    Tensor rows, cols;
    int64_t first;          // of the launch's workgroups
    int strips;             // workgroups along the columns
};
constexpr int QUANT_MAX = 3;
struct QuantArgs {
    QuantOperand o[QUANT_MAX];
    int count;
};

// By rows: 32 rows x 256 columns per workgroup; a row's 512 bytes are read by half a wave, a group's maximum is over four lanes.
// 14336 x 4096: 24 to 26 us (5.6 to 6.1 TB/s).
__global__ __launch_bounds__(THREADS) void quant_row_kernel(QuantOperand g) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t tiles = idx::mx4_tiles(g.C), tile = blockIdx.x % tiles, first = (int64_t)(blockIdx.x / tiles) * idx::MX4_ROW_BLOCK, row0 = first + (threadIdx.x >> 5);
    const int octet = threadIdx.x & 31;
    uint4 v[4];
    load_rows<4>(v, g.x, g.ldx, row0, 8, g.R, tile * idx::MX4_TILE + octet * 8, g.C, (g.C & 7) && (tile + 1) * idx::MX4_TILE > g.C);
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

// By columns (the transposed tensor's rows), with ROWS both ways from the same read, up to three tensors in a launch.  A wave has 32 rows x 512 / RB columns in
// registers, a lane 8 columns of 32 / RB rows: a column's group is RB lanes', a row's four neighbours'.  A column's codes go through LDS, from where 16 NW
// bytes of it are written in one piece.
template <int NW, int RB, bool ROWS>
__global__ __launch_bounds__(64 * NW, 4) void quant_cols_kernel(QuantArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int OCTETS = 64 / RB, COLS = OCTETS * 8, RPL = 32 / RB, ROWS_HERE = 32 * NW, GROUPS = COLS / 32, LINE = NW * 16;
    __shared__ __attribute__((aligned(16))) uint8_t lines[COLS * LINE];
    __shared__ __attribute__((aligned(16))) uint8_t row_scales[ROWS_HERE * GROUPS], col_scales[COLS * NW];
    const int64_t block = blockIdx.x;
    int which = 0;
    if (args.count > 1 && block >= args.o[1].first) which = 1;
    if (args.count > 2 && block >= args.o[2].first) which = 2;
    const QuantOperand& g = args.o[which];
    const int64_t R = g.R, C = g.C, at_block = block - g.first, chunk = at_block / g.strips, first = chunk * ROWS_HERE, col0 = (at_block - chunk * g.strips) * COLS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, octet = lane % OCTETS, part = lane / OCTETS;
    const int64_t row0 = first + wave * 32 + part * RPL;
    uint4 v[RPL];
    load_rows<RPL>(v, g.x, g.ldx, row0, 1, R, col0 + octet * 8, C, (C & 7) && col0 + COLS > C);
    const int64_t tile = col0 / idx::MX4_TILE;
    const int tile_octet = (int)(col0 % idx::MX4_TILE) / 8;
    if (ROWS) {
        uint8_t* const codes = g.rows.codes + idx::mx4_code_at(row0, g.rows.ld, tile, tile_octet + octet);
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
            const uint32_t byte = scale_byte(quad_max(halves_max(largest2(v[i]))));
            if (row0 + i < R) *reinterpret_cast<uint32_t*>(codes + i * g.rows.ld) = encode8(v[i].x, v[i].y, v[i].z, v[i].w, byte);
            if ((octet & 3) == 0) row_scales[(wave * 32 + part * RPL + i) * GROUPS + (octet >> 2)] = (uint8_t)byte;
        }
    }
    uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
        m[0] = pk_max(m[0], v[i].x & MAGNITUDE);
        m[1] = pk_max(m[1], v[i].y & MAGNITUDE);
        m[2] = pk_max(m[2], v[i].z & MAGNITUDE);
        m[3] = pk_max(m[3], v[i].w & MAGNITUDE);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (OCTETS == 8) m[j] = dpp_pk_max<0x128>(m[j]);      // (row_ror:8)
        if (OCTETS <= 16) m[j] = pk_max_16(m[j]);
        m[j] = pk_max_32(m[j]);
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const uint32_t byte = scale_byte(odd ? m[j] >> 16 : m[j] & 0xffffu);
            const auto pair = [&](int i) {      // rows i and i + 1 of this column
                const uint32_t a = j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w, b = j == 0 ? v[i + 1].x : j == 1 ? v[i + 1].y : j == 2 ? v[i + 1].z : v[i + 1].w;
                return odd ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
            };
            const int c = octet * 8 + 2 * j + odd;
            uint8_t* const to = lines + c * LINE + idx::mx4_col_chunk(wave, octet, NW) * 16 + part * (RPL / 2);
            if constexpr (RPL == 4) {
                *reinterpret_cast<uint16_t*>(to) = (uint16_t)encode4(pair(0), pair(2), byte);
            } else {
#pragma unroll
                for (int w = 0; w < RPL / 8; ++w) reinterpret_cast<uint32_t*>(to)[w] = encode8(pair(8 * w), pair(8 * w + 2), pair(8 * w + 4), pair(8 * w + 6), byte);
            }
            if (part == 0) col_scales[c * NW + wave] = (uint8_t)byte;
        }
    }
    __syncthreads();
    if (ROWS && threadIdx.x < ROWS_HERE && first + threadIdx.x < R) {
        uint8_t* const to = g.rows.scales + idx::mx4_scale_at(tile, g.rows.scale_ld, first + threadIdx.x, tile_octet / 4);
        if (GROUPS == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(row_scales + threadIdx.x * GROUPS);
        else if (GROUPS == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(row_scales + threadIdx.x * GROUPS);
        else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(row_scales + threadIdx.x * GROUPS);
    }
    const int64_t row_tile = first / idx::MX4_TILE;
    const int within = (int)(first % idx::MX4_TILE);
#pragma unroll
    for (int u = 0; u < COLS / 64; ++u) {       // NW pieces of 16 bytes to a column
        const int piece = u * 64 * NW + threadIdx.x, c = piece / NW, p = piece % NW;
        if (col0 + c < C)
            *reinterpret_cast<uint4*>(g.cols.codes + idx::mx4_code_at(col0 + c, g.cols.ld, row_tile, within / 8) + p * 16) =
                *reinterpret_cast<const uint4*>(lines + c * LINE + idx::mx4_col_chunk(p, c >> 3, NW) * 16);
    }
    for (int c = threadIdx.x; c < COLS && col0 + c < C; c += 64 * NW) {
        uint8_t* const to = g.cols.scales + idx::mx4_scale_at(row_tile, g.cols.scale_ld, col0 + c, within / 32);
        if (NW == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(col_scales + c * NW);
        else if (NW == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(col_scales + c * NW);
        else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(col_scales + c * NW);
    }
#else
    (void)args;
#endif
}

int too_many(const char* fn) { return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn); }

// Workgroups over all of x^T's tiles (those behind its last rows make the zeros up to the end of a tile) and, with them, over all columns of x
template <int NW, int RB, bool ROWS>
int launch_cols(const char* fn, QuantArgs g, hipStream_t st) {
    constexpr int COLS = 512 / RB;
    int64_t blocks = 0;
    for (int i = 0; i < g.count; ++i) {
        QuantOperand& o = g.o[i];
        o.first = blocks;
        o.strips = (int)(ROWS ? idx::mx4_tiles(o.C) * (idx::MX4_TILE / COLS) : (o.C + COLS - 1) / COLS);
        blocks += o.strips * idx::mx4_tiles(o.R) * (8 / NW);
    }
    if (!idx::grid_fits(blocks, 64 * NW)) return too_many(fn);
    quant_cols_kernel<NW, RB, ROWS><<<dim3((unsigned)blocks), dim3(64 * NW), 0, st>>>(g);
    return check_launch(fn);
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
    int once;       // whether what is read goes past the caches
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
    return v;
}

// h = bf16(x + residual), r = 1 / sqrt(mean(h^2) + eps), y = bf16(bf16(h r) w), quantised: a row in the registers of T threads (64: four rows to a workgroup),
// NV octets each.  The squares are added up in 64 bits (they are exact in it) and r is rounded to 32 once, so that an order of summation moves it by parts in 2^53 before that.  With a residual, 4 bits, tensors from memory: 1 x 4096 3.4
// us, 2047 x 4096 16.9, 16384 x 4096 84 (5.2 TB/s; a load at a time in front of a store 90); int8 by groups 2047 x 4096 17.9, 16384 x 4096 84 (5.6 TB/s).
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
    // all loads in front of the first store, which they might overlap for all that the compiler knows
    const auto load_row = [&](auto load) {
        uint4 b[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int o = t + i * T;
            v[i] = o < octets ? load(g.x + row * g.ldx + o * 8) : make_uint4(0, 0, 0, 0);
            if (g.residual && o < octets) b[i] = load(g.residual + row * g.ldr + o * 8);
        }
        if (!g.residual) return;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int o = t + i * T;
            if (o >= octets) continue;
            v[i] = make_uint4(add_bf16x2(v[i].x, b[i].x), add_bf16x2(v[i].y, b[i].y), add_bf16x2(v[i].z, b[i].z), add_bf16x2(v[i].w, b[i].w));
            *reinterpret_cast<uint4*>(g.h + row * g.ldh + o * 8) = v[i];
        }
    };
    if (g.once) load_row([](const uint16_t* p) { return load16_once(p); });
    else load_row([](const uint16_t* p) { return load16(p); });
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

// Tensors that the last-level cache does not hold beside what is written are read past the caches; smaller ones, which whoever made them has left there, are not.  us, x
// just written by another kernel, a load at a time, past them / not: 1024 x 4096 9.4 / 8.6, 2047 x 4096 17.2 / 15.6, 4096 x 4096 26.3 / 26.1, 8192 x 4096 43.7 / 48.3,
// 16384 x 4096 83.5 / 87.7.
constexpr int64_t NORM_ONCE = (int64_t)24 << 20;

int64_t norm_blocks(int64_t rows, int64_t dim) { return (rows + idx::mx4_norm_rows(dim) - 1) / idx::mx4_norm_rows(dim); }

template <int TO>
void launch_norm(NormArgs g, hipStream_t st) {
    g.once = g.rows * g.dim > NORM_ONCE;
    const int64_t blocks = norm_blocks(g.rows, g.dim);
    const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)blocks), dim3(THREADS), 0, st>>>(g); };
    static_assert(idx::mx4_norm_rows(1024) == THREADS / 64 && idx::mx4_norm_rows(1025) == 1, "a row to a wave, or to a workgroup");
    if (g.dim <= 512) go(rmsnorm_quant_kernel<64, 1, TO>);
    else if (g.dim <= 1024) go(rmsnorm_quant_kernel<64, 2, TO>);
    else if (g.dim <= 2048) go(rmsnorm_quant_kernel<THREADS, 1, TO>);
    else if (g.dim <= 4096) go(rmsnorm_quant_kernel<THREADS, 2, TO>);
    else if (g.dim <= 8192) go(rmsnorm_quant_kernel<THREADS, 4, TO>);
    else go(rmsnorm_quant_kernel<THREADS, 8, TO>);
}

}  // namespace
}  // namespace mx4
}  // namespace ti8

using namespace ti8;

extern "C" int ti8_mx4_quant(const ti8_mx4_operand* operands, int count, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_quant";
    if (!operands) return fail(TI8_ERR_NULL, "%s: operands are required", fn);
    if (count < 1 || count > mx4::QUANT_MAX) return fail(TI8_ERR_SHAPE, "%s: need 1 to %d operands, got %d", fn, mx4::QUANT_MAX, count);
    mx4::QuantArgs g;
    g.count = count;
    int64_t elements = 0;
    for (int i = 0; i < count; ++i) {
        const ti8_mx4_operand& o = operands[i];
        if (!o.x || (!o.by_rows.codes && !o.by_columns.codes)) return fail(TI8_ERR_NULL, "%s: x and one of by_rows and by_columns are required", fn);
        if (count > 1 && (!o.by_rows.codes || !o.by_columns.codes)) return fail(TI8_ERR_NULL, "%s: several operands are quantised by rows and by columns", fn);
        if (o.rows <= 0 || o.cols <= 0 || o.rows > (1 << 28) || o.cols > (1 << 28) || (o.rows > 1 && o.ldx < o.cols) || o.rows * o.cols > (1ll << 37))
            return fail(TI8_ERR_SHAPE, "%s: need rows, cols in 1 .. 2^28, up to 2^37 elements and ldx >= cols; got rows=%lld cols=%lld ldx=%lld", fn, (long long)o.rows,
                        (long long)o.cols, (long long)o.ldx);
        if (reinterpret_cast<uintptr_t>(o.x) & 1) return fail(TI8_ERR_ALIGN, "%s: x must be 2-byte aligned", fn);
        g.o[i] = {static_cast<const uint16_t*>(o.x), o.ldx, o.rows, o.cols, {}, {}, 0, 0};
        if (o.by_rows.codes)
            if (int e = mx4::check(fn, "by_rows", &o.by_rows, o.rows, o.cols, g.o[i].rows)) return e;
        if (o.by_columns.codes)
            if (int e = mx4::check(fn, "by_columns", &o.by_columns, o.cols, o.rows, g.o[i].cols)) return e;
        elements += idx::mx4_tiles(o.rows) * idx::mx4_tiles(o.cols) * idx::MX4_TILE * idx::MX4_TILE;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (!operands[0].by_columns.codes) {
        const int64_t blocks = idx::mx4_tiles(g.o[0].C) * ((g.o[0].R + idx::MX4_ROW_BLOCK - 1) / idx::MX4_ROW_BLOCK);
        if (!idx::grid_fits(blocks, mx4::THREADS)) return mx4::too_many(fn);
        mx4::quant_row_kernel<<<dim3((unsigned)blocks), dim3(mx4::THREADS), 0, st>>>(g.o[0]);
        return check_launch(fn);
    }
    // Small tensors: workgroups of 128 x 64 elements (by columns alone 64 x 64), whose code is a quarter as long (it is read from memory too); behind that twice as many
    // columns to a workgroup, whose rows' codes are written in longer pieces.  us, both ways, small / large, tensors from memory: 200 x 300 4.1 / 5.5, 1001 x 1016 4.9 / 5.3,
    // 1500 x 1500 6.3 / 8.3, 2048 x 2048 7.4 / 6.9, 4096 x 4096 17 / 16, 14336 x 4096 50 / 41 (37 since x is read past the caches: 4.9 TB/s).  By columns alone 14336 x 4096 29 (5.2 TB/s).
    const bool small = elements < (int64_t)16384 * device_cu_count(), rows = operands[0].by_rows.codes;
    if (small) return rows ? mx4::launch_cols<4, 8, true>(fn, g, st) : mx4::launch_cols<2, 8, false>(fn, g, st);
    return rows ? mx4::launch_cols<4, 4, true>(fn, g, st) : mx4::launch_cols<8, 4, false>(fn, g, st);
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
    if (!idx::grid_fits(blocks, mx4::THREADS)) return mx4::too_many(fn);
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
    if (!idx::grid_fits(blocks, mx4::THREADS)) return mx4::too_many(fn);
    mx4::dequant_row_kernel<<<dim3((unsigned)blocks), dim3(mx4::THREADS), 0, static_cast<hipStream_t>(stream)>>>(q, ldq, s, rows, cols, group ? 1 : 0, static_cast<uint16_t*>(y), ldy);
    return check_launch(fn);
}

extern "C" int ti8_rmsnorm_quant(const ti8_rmsnorm_quant_args* a, ti8_stream_t stream) {
    const char* const fn = "ti8_rmsnorm_quant";
    if (!a || !a->x || !a->w || !a->rstd) return fail(TI8_ERR_NULL, "%s: x, w and rstd are required", fn);
    if (!a->residual != !a->h) return fail(TI8_ERR_NULL, "%s: residual and h go together", fn);
    if (!a->mx4.codes == !a->q) return fail(TI8_ERR_NULL, "%s: one of mx4 and q is required", fn);
    const int64_t rows = a->rows, dim = a->dim;
    if (rows <= 0 || dim <= 0 || dim % 8 || dim > mx4::NORM_MAX_DIM || a->ldx < dim || (a->residual && (a->ldr < dim || a->ldh < dim)))
        return fail(TI8_ERR_SHAPE, "%s: need rows, dim a multiple of 8 up to %d and leading dimensions of at least dim; got rows=%lld dim=%lld", fn, mx4::NORM_MAX_DIM,
                    (long long)rows, (long long)dim);
    if (rows > (1 << 28) || !idx::grid_fits(mx4::norm_blocks(rows, dim), mx4::THREADS))
        return fail(TI8_ERR_SHAPE, "%s: up to 2^26 - 4 rows, of more than 1024 elements up to 2^24 - 1; got rows=%lld dim=%lld", fn, (long long)rows, (long long)dim);
    if (!aligned16(a->x) || !aligned16(a->w) || !aligned16(a->residual) || !aligned16(a->h) || a->ldx % 8 || (a->residual && (a->ldr % 8 || a->ldh % 8)) ||
        (reinterpret_cast<uintptr_t>(a->rstd) & 3))
        return fail(TI8_ERR_ALIGN, "%s: rows of x, residual and h and the weight must be 16-byte aligned", fn);
    mx4::NormArgs g{static_cast<const uint16_t*>(a->x), static_cast<const uint16_t*>(a->residual), static_cast<const uint16_t*>(a->w), a->ldx, a->ldr, a->ldh, rows,
                    static_cast<uint16_t*>(a->h), a->rstd, (int)dim, a->eps, {}, a->q, a->ldq, a->s, {}, 0};
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
