// C = A B^T of two tensors in 4 bits with shared scales (format: mx4.h) on v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies the codes, applies both
// operands' scales and adds up in fp32; C is rounded once.
//
// A K tile is 256 elements: 128 bytes of codes per row, staged in LDS by direct loads (16-byte chunks XOR-swizzled by row, so that the 16 rows a quarter
// of a wave reads at one chunk lie in distinct banks), double buffered, and 8 scales per row, which go straight into registers.  Lane l of an instruction
// supplies row l % 32 of its operand and 32 elements of the 64 that it contracts.  Which 32 is free as long as both operands agree: step ks of a tile takes
// chunk ks from lanes below 32 and chunk 4 + ks from the others, so that a lane's four scales of a tile are one word, and the step's number picks the byte.
// The operands change places (the instruction's rows are C's columns), so that a lane holds four neighbouring elements of a row of C.
#include "mx4.h"

namespace ti8 {
namespace mx4 {
namespace {

struct Gemm {
    const uint8_t *A, *B, *SA, *SB;
    void* C;
    int64_t lda, ldb, sla, slb;         // bytes between rows, between tiles of scales
    int64_t rows_a, rows_b;             // rows between batches
    int64_t ldc, bsc;
    int M, N, nk, tiles_m, tiles_n, wide;
};

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

template <int KS>
__device__ __forceinline__ v16f multiply(const v4i& b, const v4i& a, const v16f& c, int sb, int sa) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1),
                                                           __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), c, 4, 4, KS, sb, KS, sa);
#else
    (void)b; (void)a; (void)sb; (void)sa;
    return c;
#endif
}

// One BM x BN tile of C on WM x WN waves
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 1) void gemm_kernel(Gemm g) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int A_INSTR = BM / 8 / NW, B_INSTR = BN / 8 / NW, A_BYTES = BM * 128, B_BYTES = BN * 128;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    uint8_t* const ldsA = smem;
    uint8_t* const ldsB = smem + 2 * A_BYTES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const idx::TileCoord tc = idx::gemm_tile_of(blockIdx.x, g.tiles_m, g.tiles_n, idx::gemm_group_rows(BM), false);
    const int m0 = tc.tile_m * BM, n0 = tc.tile_n * BN;
    const int64_t first_a = blockIdx.z * g.rows_a + m0, first_b = blockIdx.z * g.rows_b + n0;
    const int rows_a = min(g.M - m0, BM), rows_b = min(g.N - n0, BN);

    // global -> LDS: an instruction of a wave covers 8 rows, lane l lands at byte 16 l of them; rows beyond the operand repeat its last
    const uint8_t *at_a = g.A + first_a * g.lda, *at_b = g.B + first_b * g.ldb;
    uint32_t off_a[A_INSTR], off_b[B_INSTR];
#pragma unroll
    for (int i = 0; i < A_INSTR; ++i) {
        const int r = (wave * A_INSTR + i) * 8 + (lane >> 3);
        off_a[i] = (uint32_t)(idx::mx4_row(r, rows_a) * (int)g.lda) + (((uint32_t)(lane & 7) ^ idx::mx4_chunk_swizzle(r)) * 16);
    }
#pragma unroll
    for (int i = 0; i < B_INSTR; ++i) {
        const int r = (wave * B_INSTR + i) * 8 + (lane >> 3);
        off_b[i] = (uint32_t)(idx::mx4_row(r, rows_b) * (int)g.ldb) + (((uint32_t)(lane & 7) ^ idx::mx4_chunk_swizzle(r)) * 16);
    }
    const auto issue = [&](int kt, int buf) {
        const uint8_t *a = at_a + (int64_t)kt * 128, *b = at_b + (int64_t)kt * 128;
#pragma unroll
        for (int i = 0; i < A_INSTR; ++i) {
            uint32_t o = off_a[i];
            asm volatile("" : "+v"(o));
            __builtin_amdgcn_global_load_lds(a + o, ldsA + buf * A_BYTES + (wave * A_INSTR + i) * 1024, 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < B_INSTR; ++i) {
            uint32_t o = off_b[i];
            asm volatile("" : "+v"(o));
            __builtin_amdgcn_global_load_lds(b + o, ldsB + buf * B_BYTES + (wave * B_INSTR + i) * 1024, 16, 0, 0);
        }
    };

    // LDS -> registers
    const int row = lane & 31, half = lane >> 5;
    const uint32_t sw = idx::mx4_chunk_swizzle(lane);
    uint32_t chunk[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) chunk[ks] = ((half * 4 + ks) ^ sw) * 16;
    const uint8_t *frag_a = ldsA + (wm * TM * 32 + row) * 128, *frag_b = ldsB + (wn * TN * 32 + row) * 128;
    const uint8_t *scales_a = g.SA + first_a * 8, *scales_b = g.SB + first_b * 8;
    uint32_t soff_a[TM], soff_b[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) soff_a[i] = idx::mx4_row((wm * TM + i) * 32 + row, rows_a) * 8 + half * 4;
#pragma unroll
    for (int j = 0; j < TN; ++j) soff_b[j] = idx::mx4_row((wn * TN + j) * 32 + row, rows_b) * 8 + half * 4;

    v16f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    v4i a[2][TM], b[2][TN];
    int sa[TM], sb[TN], na[TM], nb[TN];
    const auto frags = [&](int set, int buf, int ks) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a[set][i] = *reinterpret_cast<const v4i*>(frag_a + buf * A_BYTES + i * 4096 + chunk[ks]);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[set][j] = *reinterpret_cast<const v4i*>(frag_b + buf * B_BYTES + j * 4096 + chunk[ks]);
    };
    const auto scales = [&](int kt) {
        const uint8_t *pa = scales_a + kt * g.sla, *pb = scales_b + kt * g.slb;
#pragma unroll
        for (int i = 0; i < TM; ++i) na[i] = *reinterpret_cast<const int*>(pa + soff_a[i]);
#pragma unroll
        for (int j = 0; j < TN; ++j) nb[j] = *reinterpret_cast<const int*>(pb + soff_b[j]);
    };

    const int last = g.nk - 1;
    scales(0);
    issue(0, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    issue(min(1, last), 1);
    frags(0, 0, 0);
    for (int kt = 0; kt <= last; ++kt) {
        const int cur = kt & 1;
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = na[i];
#pragma unroll
        for (int j = 0; j < TN; ++j) sb[j] = nb[j];
        scales(min(kt + 1, last));
#define TI8_STEP(KS)                                                                                                          \
    _Pragma("unroll") for (int i = 0; i < TM; ++i) _Pragma("unroll") for (int j = 0; j < TN; ++j) acc[i][j] =                 \
        multiply<KS>(b[KS & 1][j], a[KS & 1][i], acc[i][j], sb[j], sa[i]);
        frags(1, cur, 1);
        TI8_STEP(0)
        frags(0, cur, 2);
        TI8_STEP(1)
        frags(1, cur, 3);
        TI8_STEP(2)
        // the next tile and its scales are there, and nobody reads this one any more (its last fragments are in registers)
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        issue(min(kt + 2, last), cur);
        frags(0, cur ^ 1, 0);
        TI8_STEP(3)
#undef TI8_STEP
    }
    __builtin_amdgcn_s_waitcnt(0);      // (loads past the last tile, repeated into LDS)
    __syncthreads();

    // lane: row m = l % 32 of a 32 x 32 block of C, columns 8 (r / 4) + 4 (l / 32) + r % 4
    const int cols = g.N - n0 - wn * TN * 32;
    if (g.wide) {
        float* const C = static_cast<float*>(g.C) + blockIdx.z * g.bsc + n0 + wn * TN * 32;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + (wm * TM + i) * 32 + row;
            if (m >= g.M) continue;
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = j * 32 + 8 * q + 4 * half;
                    float* const to = C + m * g.ldc + n;
                    if (n + 4 <= cols) {
                        typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
                        *reinterpret_cast<v4f_any*>(to) = v4f{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (n + c < cols) to[c] = acc[i][j][4 * q + c];
                    }
                }
        }
        return;
    }
    // through LDS, a wave's 32 rows at a time, so that a row is written in one piece
    constexpr int WIDTH = TN * 32, PITCH = WIDTH * 2 + 16, LPR = WIDTH / 8, RPI = 64 / LPR;
    static_assert(32 * PITCH * NW <= 2 * (A_BYTES + B_BYTES), "the waves' rows fit the operands' buffers");
    uint8_t* const mine = smem + wave * 32 * PITCH;
    uint16_t* const C = static_cast<uint16_t*>(g.C) + blockIdx.z * g.bsc + n0 + wn * WIDTH;
    const int n = (lane % LPR) * 8;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint2*>(mine + row * PITCH + (j * 32 + 8 * q + 4 * half) * 2) =
                    make_uint2(pack_bf16x2(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack_bf16x2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]));
#pragma unroll
        for (int u = 0; u < 32 / RPI; ++u) {
            const int r = u * RPI + lane / LPR, m = m0 + (wm * TM + i) * 32 + r;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + r * PITCH + n * 2);
            if (m < g.M) store8(C + m * g.ldc + n, v, cols - n);
        }
    }
#else
    (void)g;
#endif
}

template <int BM, int BN, int WM, int WN>
int launch(const char* fn, Gemm g, int64_t batch, hipStream_t st) {
    constexpr int LDS = 2 * (BM + BN) * 128;
    static OncePerDevice once;
    const auto kernel = gemm_kernel<BM, BN, WM, WN>;
    if (LDS > 65536 && raise_lds_limit(once, reinterpret_cast<const void*>(kernel), LDS) != hipSuccess) return fail(TI8_ERR_HIP, "%s: %d bytes of LDS refused", fn, LDS);
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    if ((int64_t)g.tiles_m * g.tiles_n > 0x7fffffff) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    kernel<<<dim3((unsigned)(g.tiles_m * g.tiles_n), 1, (unsigned)batch), dim3(64 * WM * WN), LDS, st>>>(g);
    return check_launch(fn);
}

}  // namespace
}  // namespace mx4
}  // namespace ti8

using namespace ti8;

extern "C" int ti8_mx4_gemm_nt(const ti8_mx4* a, int64_t rows_a, const ti8_mx4* b, int64_t rows_b, void* c, int64_t ldc, int64_t bsc, int64_t batch, int64_t M, int64_t N,
                               int64_t K, int wide, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_gemm_nt";
    if (!a || !b || !c) return fail(TI8_ERR_NULL, "%s: a, b and c are required", fn);
    if (M <= 0 || N <= 0 || K <= 0 || batch <= 0 || batch > 65535 || M > (1 << 28) || N > (1 << 28) || K > (1 << 22) || ldc < N || bsc < 0 || (rows_a != 0 && rows_a < M) ||
        (rows_b != 0 && rows_b < N))
        return fail(TI8_ERR_SHAPE, "%s: need M, N in 1 .. 2^28, K in 1 .. 2^22, batch in 1 .. 65535, ldc >= N and batches of as many rows; got M=%lld N=%lld K=%lld batch=%lld ldc=%lld "
                    "rows_a=%lld rows_b=%lld", fn, (long long)M, (long long)N, (long long)K, (long long)batch, (long long)ldc, (long long)rows_a, (long long)rows_b);
    // (the last row that any batch reads)
    mx4::Tensor ta, tb;
    if (int e = mx4::check(fn, "a", a, (batch - 1) * rows_a + M, K, ta)) return e;
    if (int e = mx4::check(fn, "b", b, (batch - 1) * rows_b + N, K, tb)) return e;
    if (ta.ld > (1 << 22) || tb.ld > (1 << 22)) return fail(TI8_ERR_SHAPE, "%s: rows of codes may be up to 2^22 bytes apart", fn);
    if (reinterpret_cast<uintptr_t>(c) & (wide ? 3 : 1)) return fail(TI8_ERR_ALIGN, "%s: c must be aligned to its elements", fn);
    const mx4::Gemm g{ta.codes, tb.codes, ta.scales, tb.scales, c, ta.ld, tb.ld, ta.scale_ld, tb.scale_ld, rows_a, rows_b, ldc, bsc, (int)M, (int)N, (int)idx::mx4_tiles(K), 0, 0, wide ? 1 : 0};
    return mx4::launch<128, 128, 2, 2>(fn, g, batch, static_cast<hipStream_t>(stream));
}
