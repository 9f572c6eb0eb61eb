// C = A B^T of two tensors in 4 bits with shared scales (format: mx4.h) on v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies the codes, applies both
// operands' scales and adds up in fp32; C is rounded once.
//
// A K tile is 256 elements: 128 bytes of codes per row, staged in LDS by direct loads (16-byte chunks XOR-swizzled by row, so that the 16 rows a quarter
// of a wave reads at one chunk lie in distinct banks), two to four tiles of them, and 8 scales per row, which go the same way (a ring of four or eight).  Lane l of an instruction
// supplies row l % 32 of its operand and 32 elements of the 64 that it contracts.  Which 32 is free as long as both operands agree: step ks of a tile takes
// chunk ks from lanes below 32 and chunk 4 + ks from the others, so that a lane's four scales of a tile are one word, and the step's number picks the byte.
// The operands change places (the instruction's rows are C's columns), so that a lane holds four neighbouring elements of a row of C.
#include <type_traits>
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
    int parts;                          // workgroups that share the contraction of a tile: C is then fp32, one after the other `part` elements apart
    int64_t part;
};

// Up to three products of a launch: number i has the workgroups from first[i] on (multiples of 8: workgroups go round the XCDs)
constexpr int TOGETHER = 3;
struct Gemms {
    Gemm g[TOGETHER];
    int first[TOGETHER + 1], count;
};

// This workgroup's product, and its number there.  A launch of one product is a kernel of its own: looking the product up takes 0.6 us before the first load
// (16 x 4096 x 4096 5.0 us / 4.5, 128 x 4096 x 4096 7.7 / 7.2).
__device__ __forceinline__ const Gemm& product_of(const Gemm& g, int& block) {
    block = blockIdx.x;
    return g;
}
__device__ __forceinline__ const Gemm& product_of(const Gemms& all, int& block) {
    const int which = idx::gemm_multi_pick(blockIdx.x, all.first[1], all.first[2], all.count);
    block = blockIdx.x - all.first[which];
    return all.g[which];
}

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

// Order of one step of a K tile: one LDS read and one load from memory, while there are any, behind each matrix instruction; nothing of another step among them.
// (Left to itself the compiler reads a step's fragments right before it needs them: 8192 x 14336 x 4096 243 us.)
template <int NMFMA, int NDS, int NVM>
__device__ __forceinline__ void interleave() {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int DS = (NDS + NMFMA - 1) / NMFMA, VM = (NVM + NMFMA - 1) / NMFMA;
#pragma unroll
    for (int q = 0; q < NMFMA; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (q * DS < NDS) __builtin_amdgcn_sched_group_barrier(0x100, DS, 0);
        if (q * VM < NVM) __builtin_amdgcn_sched_group_barrier(0x020, VM, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#endif
}

// What of n pieces of work goes beside matrix instruction q of `count`: f(i) for its share
template <class F>
__device__ __forceinline__ void beside(int q, int count, int n, const F& f) {
#pragma unroll
    for (int i = 0; i < n; ++i)
        if (i >= q * n / count && i < (q + 1) * n / count) f(i);
}

// One BM x BN tile of C on WM x WN waves, with STAGES tiles of codes in LDS.  256 x 256, 8192 x 14336 x 4096: 220 to 235 us (4.1 to 4.4 PFLOP/s).  A K tile takes 3520
// cycles of a CU in all, of which the matrix pipe has 2048 (0.58) and LDS 1180 (0.17 of them conflicts); 4 to 5 us of each round of tiles are first loads and results,
// the rest is the one barrier per tile, behind which all eight waves read at once.  On codes of zero the cycles are the same, at 2.16 GHz instead of 1.76: power sets the
// clock (a loop of nothing but these instructions reaches 6.5 PFLOP/s on random codes, 9.8 on zeros), not the cycles without the pipe.  16 x 16 x 128 instructions (their
// loop: 7.2 and 9.7), four waves of 128 x 128, workgroups that go on to the next tile: within 3 %.  Smaller tiles where those do not fill the CUs: 700 x 4096 x 4096 10.3
// to 11.5 us, 128 x 4096 x 4096 5.9, of which 2.2 are the launch and 1.5 to 3 a tile's first loads and results.
constexpr int scale_stages(int stages) { return stages == 2 ? 4 : 8; }
constexpr int gemm_lds(int bm, int bn, int stages) { return (bm + bn) * (128 * stages + 8 * scale_stages(stages)); }
constexpr int waitcnt(int vm, int other) { return ((vm >> 4) << 14) | (vm & 15) | other; }      // vmcnt[3:0] | expcnt << 4 | lgkmcnt << 8 | vmcnt[5:4] << 14

template <int BM, int BN, int WM, int WN, int STAGES, class Products>
__global__ __launch_bounds__(64 * WM * WN, 1) void gemm_kernel(Products products) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool MANY = std::is_same<Products, Gemms>::value;
    int block;
    const Gemm& g = product_of(products, block);
    if (MANY && block >= g.tiles_m * g.tiles_n) return;
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int A_INSTR = BM / 8 / NW, B_INSTR = BN / 8 / NW, A_BYTES = BM * 128, B_BYTES = BN * 128;
    constexpr int SA_INSTR = (BM / 32 + NW - 1) / NW, SB_INSTR = (BN / 32 + NW - 1) / NW, S_BYTES = (BM + BN) * 8, RING = scale_stages(STAGES);
    constexpr bool WHOLE = TM * TN <= 4;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    uint8_t* const ldsA = smem;
    uint8_t* const ldsB = smem + STAGES * A_BYTES;
    uint8_t* const ldsS = ldsB + STAGES * B_BYTES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const idx::TileCoord tc = idx::gemm_tile_of(block, g.tiles_m, g.tiles_n, idx::gemm_group_rows(BM), MANY);
    const int m0 = tc.tile_m * BM, n0 = tc.tile_n * BN;
    const int64_t first_a = blockIdx.z * g.rows_a + m0, first_b = blockIdx.z * g.rows_b + n0;
    const int rows_a = min(g.M - m0, BM), rows_b = min(g.N - n0, BN);

    const idx::Mx4Part part = idx::mx4_part(blockIdx.y, g.parts, g.nk);
    const int last = part.tiles - 1;
    // global -> LDS: an instruction of a wave covers 8 rows, lane l lands at byte 16 l of them; rows beyond the operand repeat its last
    const uint8_t *at_a = g.A + first_a * g.lda + part.first * 128, *at_b = g.B + first_b * g.ldb + part.first * 128;
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
    constexpr int LOADS = A_INSTR + B_INSTR, FIRST = LOADS / 2;
    const auto issue = [&](int kt, int stage, int from, int to) {
        const uint8_t *a = at_a + (int64_t)min(kt, last) * 128, *b = at_b + (int64_t)min(kt, last) * 128;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (i < from || i >= to) continue;
            const bool of_a = i < A_INSTR;
            uint32_t o = of_a ? off_a[of_a ? i : 0] : off_b[of_a ? 0 : i - A_INSTR];
            asm volatile("" : "+v"(o));     // (a uniform address and a 32-bit offset, not a sum in 64 bits)
            if (of_a) __builtin_amdgcn_global_load_lds(a + o, ldsA + stage * A_BYTES + (wave * A_INSTR + i) * 1024, 16, 0, 0);
            else __builtin_amdgcn_global_load_lds(b + o, ldsB + stage * B_BYTES + (wave * B_INSTR + i - A_INSTR) * 1024, 16, 0, 0);
        }
    };
    // scales of a tile: 32 rows to an instruction, lane l lands at byte 4 l of their 256
    const uint8_t *scales_a = g.SA + first_a * 8 + part.first * g.sla, *scales_b = g.SB + first_b * 8 + part.first * g.slb;
    uint32_t soff_a[SA_INSTR], soff_b[SB_INSTR];
#pragma unroll
    for (int i = 0; i < SA_INSTR; ++i) soff_a[i] = idx::mx4_row((wave + i * NW) % (BM / 32) * 32 + (lane >> 1), rows_a) * 8 + (lane & 1) * 4;
#pragma unroll
    for (int i = 0; i < SB_INSTR; ++i) soff_b[i] = idx::mx4_row((wave + i * NW) % (BN / 32) * 32 + (lane >> 1), rows_b) * 8 + (lane & 1) * 4;
    constexpr int SCALE_LOADS = SA_INSTR + SB_INSTR;
    const auto issue_scale = [&](int kt, int i) {
        const bool of_a = i < SA_INSTR;
        const uint8_t* const from = of_a ? scales_a + min(kt, last) * g.sla : scales_b + min(kt, last) * g.slb;
        uint32_t o = of_a ? soff_a[of_a ? i : 0] : soff_b[of_a ? 0 : i - SA_INSTR];
        asm volatile("" : "+v"(o));
        __builtin_amdgcn_global_load_lds(from + o, ldsS + kt % RING * S_BYTES + (of_a ? (wave + i * NW) % (BM / 32) * 256 : BM * 8 + (wave + (i - SA_INSTR) * NW) % (BN / 32) * 256), 4, 0, 0);
    };
    const auto issue_scales = [&](int kt) {
#pragma unroll
        for (int i = 0; i < SCALE_LOADS; ++i) issue_scale(kt, i);
    };

    // LDS -> registers
    const int row = lane & 31, half = lane >> 5;
    const uint32_t sw = idx::mx4_chunk_swizzle(lane);
    uint32_t chunk[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) chunk[ks] = ((half * 4 + ks) ^ sw) * 16;
    const uint8_t *frag_a = ldsA + (wm * TM * 32 + row) * 128, *frag_b = ldsB + (wn * TN * 32 + row) * 128;
    const uint8_t *scale_a = ldsS + (wm * TM * 32 + row) * 8 + half * 4, *scale_b = ldsS + BM * 8 + (wn * TN * 32 + row) * 8 + half * 4;

    v16f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    v4i a[2][TM], b[2][TN];
    int sa[TM], sb[TN], na[TM], nb[TN];
    const auto frags = [&](int set, int stage, int ks) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a[set][i] = *reinterpret_cast<const v4i*>(frag_a + stage * A_BYTES + i * 4096 + chunk[ks]);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[set][j] = *reinterpret_cast<const v4i*>(frag_b + stage * B_BYTES + j * 4096 + chunk[ks]);
    };
    const auto scales = [&](int kt) {
#pragma unroll
        for (int i = 0; i < TM; ++i) na[i] = *reinterpret_cast<const int*>(scale_a + kt % RING * S_BYTES + i * 256);
#pragma unroll
        for (int j = 0; j < TN; ++j) nb[j] = *reinterpret_cast<const int*>(scale_b + kt % RING * S_BYTES + j * 256);
    };

    if constexpr (WHOLE) {
        // All of the next tile's fragments are read beside this one's matrix instructions, and tile kt + STAGES asked for (everybody has tile kt in registers), a piece
        // of both behind each instruction and in this order: left to the compiler they come in bunches, and LDS and the matrix pipe take turns (512 x 4096 x 4096
        // 12.4 us on 128 x 128, 10.8 on 64 x 64, so 11.2 and 10.1).  (256 x 256 is no faster with it.)
        constexpr int BEHIND = (STAGES - 2) * (LOADS + SCALE_LOADS);
        static_assert((STAGES - 1) * (LOADS + SCALE_LOADS) < 64 && RING >= STAGES, "vmcnt has six bits");
        v4i wa[2][TM][4], wb[2][TN][4];
        int ws[2][TM], wt[2][TN];
        constexpr int FRAGS = 4 * (TM + TN), STEPS = 4 * TM * TN;
        const auto read_scale = [&](int set, int kt, int i) {
            if (i < TM) ws[set][i < TM ? i : 0] = *reinterpret_cast<const int*>(scale_a + kt % RING * S_BYTES + i * 256);
            else wt[set][i < TM ? 0 : i - TM] = *reinterpret_cast<const int*>(scale_b + kt % RING * S_BYTES + (i - TM) * 256);
        };
        const auto read = [&](int set, int stage, int i) {
            const int ks = i / (TM + TN), x = i % (TM + TN);
            if (x < TM) wa[set][x < TM ? x : 0][ks] = *reinterpret_cast<const v4i*>(frag_a + stage * A_BYTES + x * 4096 + chunk[ks]);
            else wb[set][x < TM ? 0 : x - TM][ks] = *reinterpret_cast<const v4i*>(frag_b + stage * B_BYTES + (x - TM) * 4096 + chunk[ks]);
        };
#pragma unroll
        for (int t = 0; t < STAGES; ++t) {
            issue(t, t, 0, LOADS);
            issue_scales(t);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(waitcnt((STAGES - 1) * (LOADS + SCALE_LOADS), 0x70));
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) read_scale(0, 0, i);
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) read(0, 0, i);
        int cur = 0, kt = 0;
#define TI8_STEP(KS, SET)                                                                                                     \
    _Pragma("unroll") for (int i = 0; i < TM; ++i) _Pragma("unroll") for (int j = 0; j < TN; ++j) {                           \
        const int q = KS * TM * TN + i * TN + j;                                                                              \
        acc[i][j] = multiply<KS>(wb[SET][j][KS], wa[SET][i][KS], acc[i][j], wt[SET][j], ws[SET][i]);                          \
        beside(q, STEPS, FRAGS, [&](int x) { read(1 - SET, next, x); });                                                      \
        if (q == 0) _Pragma("unroll") for (int x = 0; x < TM + TN; ++x) read_scale(1 - SET, kt + 1, x);                       \
        beside(q, STEPS, LOADS, [&](int x) { issue(kt + STAGES, cur, x, x + 1); });                                           \
        beside(q, STEPS, SCALE_LOADS, [&](int x) { issue_scale(kt + STAGES, x); });                                           \
        __builtin_amdgcn_sched_barrier(0);                                                                                    \
    }
#define TI8_TILE(SET)                                                                                                         \
    {                                                                                                                         \
        const int next = cur + 1 == STAGES ? 0 : cur + 1;                                                                     \
        __builtin_amdgcn_s_waitcnt(waitcnt(BEHIND, 0x70));                                                                    \
        asm volatile("s_barrier" ::: "memory");                                                                               \
        TI8_STEP(0, SET) TI8_STEP(1, SET) TI8_STEP(2, SET) TI8_STEP(3, SET)                                                   \
        cur = next;                                                                                                           \
        ++kt;                                                                                                                 \
    }
        for (;;) {
            TI8_TILE(0)
            if (kt > last) break;
            TI8_TILE(1)
            if (kt > last) break;
        }
#undef TI8_TILE
#undef TI8_STEP
    } else {
        // Codes of tile kt + STAGES are asked for once tile kt has been read, half of them a step later, scales of tile kt + STAGES + 1 before that (and so in front of the
        // loop: what is waited for is counted from the end).  (Loads past the last tile repeat it: no branches in the loop.)
        constexpr int BEHIND = idx::mx4_behind(STAGES, LOADS, SCALE_LOADS);
        static_assert(BEHIND + FIRST < 64, "vmcnt has six bits");
        issue_scales(0);
        issue_scales(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t) {
            issue(t, t, 0, LOADS);
            __builtin_amdgcn_sched_barrier(0);
            issue_scales(t + 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        issue(STAGES - 1, STAGES - 1, 0, FIRST);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(waitcnt(BEHIND + FIRST, 0x70));
        asm volatile("s_barrier" ::: "memory");
        frags(0, 0, 0);
        scales(0);
        int cur = 0, fill = STAGES - 1;       // stages of tile kt and of the one that is being fetched
        for (int kt = 0; kt <= last; ++kt) {
            const int next = cur + 1 == STAGES ? 0 : cur + 1;
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[i] = na[i];
#pragma unroll
            for (int j = 0; j < TN; ++j) sb[j] = nb[j];
#define TI8_STEP(KS)                                                                                                          \
        _Pragma("unroll") for (int i = 0; i < TM; ++i) _Pragma("unroll") for (int j = 0; j < TN; ++j) acc[i][j] =                 \
            multiply<KS>(b[KS & 1][j], a[KS & 1][i], acc[i][j], sb[j], sa[i]);
            frags(1, cur, 1);
            issue(kt + STAGES - 1, fill, FIRST, LOADS);
            TI8_STEP(0)
            interleave<TM * TN, TM + TN, LOADS - FIRST>();
            frags(0, cur, 2);
            issue_scales(kt + STAGES + 1);
            TI8_STEP(1)
            interleave<TM * TN, TM + TN, SCALE_LOADS>();
            frags(1, cur, 3);
            TI8_STEP(2)
            interleave<TM * TN, TM + TN, 0>();
            // the next tile is there, and nobody reads this one any more (its last fragments are in registers)
            __builtin_amdgcn_s_waitcnt(waitcnt(BEHIND, 0x70));       // lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");                  // (not __syncthreads(), which would wait for all loads)
            issue(kt + STAGES, cur, 0, FIRST);
            frags(0, next, 0);
            scales(kt + 1);
            TI8_STEP(3)
            interleave<TM * TN, 2 * (TM + TN), FIRST>();
#undef TI8_STEP
            fill = cur;
            cur = next;
        }
    }
    __builtin_amdgcn_s_waitcnt(0);      // (loads past the last tile, repeated into LDS)
    __syncthreads();

    // Lane: row m = l % 32 of a 32 x 32 block of C, columns 8 q + 4 (l / 32) + c in register 4 q + c.  Through LDS, 32 rows of a wave's at a time, so that a row is
    // written in one piece
    const int64_t first_c = blockIdx.y * g.part + blockIdx.z * g.bsc + (int64_t)(m0 + wm * TM * 32) * g.ldc + n0 + wn * TN * 32;
    const int rows_left = g.M - m0 - wm * TM * 32, cols_left = g.N - n0 - wn * TN * 32;
    const auto write = [&](auto wide, auto put) {
        constexpr int SIZE = decltype(wide)::value ? 4 : 2, WIDTH = TN * 32, PITCH = WIDTH * SIZE + 16, PER = 16 / SIZE, LPR = WIDTH / PER, RPI = 64 / LPR;
        static_assert(32 * PITCH * NW <= STAGES * (A_BYTES + B_BYTES), "the waves' rows fit the operands' buffers");
        uint8_t* const mine = smem + wave * 32 * PITCH;
        const int n = (lane % LPR) * PER;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint8_t* const to = mine + row * PITCH + (j * 32 + 8 * q + 4 * half) * SIZE;
                    const v4f x = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if constexpr (SIZE == 4) *reinterpret_cast<v4f*>(to) = x;
                    else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
                }
#pragma unroll
            for (int u = 0; u < 32 / RPI; ++u) {
                const int r = u * RPI + lane / LPR;
                const uint4 v = *reinterpret_cast<const uint4*>(mine + r * PITCH + n * SIZE);
                if (i * 32 + r < rows_left) put(first_c + (i * 32 + r) * g.ldc + n, v, cols_left - n);
            }
        }
    };
    if (g.wide)
        write(std::true_type(), [&](int64_t at, const uint4& v, int left) {
            typedef u32x4 u32x4_word __attribute__((aligned(4)));
            uint32_t* const to = static_cast<uint32_t*>(g.C) + at;
            if (left >= 4) {
                *reinterpret_cast<u32x4_word*>(to) = __builtin_bit_cast(u32x4, v);
            } else {
                if (left > 0) to[0] = v.x;
                if (left > 1) to[1] = v.y;
                if (left > 2) to[2] = v.z;
            }
        });
    else
        // Results of the largest tiles go past the caches, which keep the operands: 16384 x 4096 x 1024 72 us / 56 (with a kernel behind it that reads C 109 / 87),
        // 8192 x 14336 x 4096 with a reader 279 / 273, 4096 x 4096 x 4096 43.6 / 43.8.  (128 x 128, 16384 x 4096 x 1024: 58 / 61.)
        write(std::false_type(), [&](int64_t at, const uint4& v, int left) {
            uint16_t* const to = static_cast<uint16_t*>(g.C) + at;
            if (BM == 256 && left >= 8) stream16(to, v);
            else store8(to, v, left);
        });
#else
    (void)products;
#endif
}

// Few rows of A: the weight passes once from memory straight into registers.  A workgroup has 16 NB rows of B and 16 MB of A, its waves take turns at the K
// tiles and add up their parts in LDS, in order.  v_mfma_scale_f32_16x16x128_f8f6f4: lane l supplies row l % 16 and 32 of 128 elements, chunk l / 16 of each half
// of a tile, so that four lanes read 64 bytes of a row in one piece.
__device__ __forceinline__ v4f multiply16(const v4i& b, const v4i& a, const v4f& c, int sb, int sa) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1),
                                                            __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), c, 4, 4, 0, sb, 0, sa);
#else
    (void)b; (void)a; (void)sb; (void)sa;
    return c;
#endif
}

template <int MB, int NB, int NW, class Products>
__global__ __launch_bounds__(64 * NW) void few_rows_kernel(Products products) {
#if defined(__HIP_DEVICE_COMPILE__)
    int block;
    const Gemm& g = product_of(products, block);
    constexpr int BLOCK = MB * NB * 256;        // elements of C here
    extern __shared__ __attribute__((aligned(16))) float parts[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, q = lane >> 4;
    const int n0 = block * (16 * NB), m0 = blockIdx.y * (16 * MB);
    if (n0 >= g.N || m0 >= g.M) return;
    const int64_t first_a = blockIdx.z * g.rows_a + m0, first_b = blockIdx.z * g.rows_b + n0;
    const uint8_t *pa[MB], *pb[NB], *qa[MB], *qb[NB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int64_t r = first_a + idx::mx4_row(i * 16 + row, g.M - m0);
        pa[i] = g.A + r * g.lda + q * 16;
        qa[i] = g.SA + r * 8;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int64_t r = first_b + idx::mx4_row(j * 16 + row, g.N - n0);
        pb[j] = g.B + r * g.ldb + q * 16;
        qb[j] = g.SB + r * 8;
    }
    struct Set {
        v4i a[MB][2], b[NB][2];
        uint2 sa[MB], sb[NB];
    };
    const auto load = [&](Set& s, int kt) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            s.b[j][0] = *reinterpret_cast<const v4i*>(pb[j] + kt * 128);
            s.b[j][1] = *reinterpret_cast<const v4i*>(pb[j] + kt * 128 + 64);
            s.sb[j] = *reinterpret_cast<const uint2*>(qb[j] + kt * g.slb);
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            s.a[i][0] = *reinterpret_cast<const v4i*>(pa[i] + kt * 128);
            s.a[i][1] = *reinterpret_cast<const v4i*>(pa[i] + kt * 128 + 64);
            s.sa[i] = *reinterpret_cast<const uint2*>(qa[i] + kt * g.sla);
        }
    };
    v4f acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const auto product = [&](const Set& s) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = multiply16(s.b[j][0], s.a[i][0], acc[i][j], s.sb[j].x >> (8 * q), s.sa[i].x >> (8 * q));
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = multiply16(s.b[j][1], s.a[i][1], acc[i][j], s.sb[j].y >> (8 * q), s.sa[i].y >> (8 * q));
    };
    // two tiles of a wave on their way at a time
    Set even, odd;
    int kt = wave;
    if (kt < g.nk) load(even, kt);
    while (kt < g.nk) {
        if (kt + NW < g.nk) load(odd, kt + NW);
        product(even);
        kt += NW;
        if (kt >= g.nk) break;
        if (kt + NW < g.nk) load(even, kt + NW);
        product(odd);
        kt += NW;
    }
    // lane: row m = l % 16 of a 16 x 16 block of C, columns 4 (l / 16) .. + 3: blocks of C in LDS as [wave][i][m][16 NB columns]
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<v4f*>(parts + wave * BLOCK + (i * 16 + row) * (16 * NB) + j * 16 + q * 4) = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x * 4; e < BLOCK; e += 64 * NW * 4) {
        v4f sum = *reinterpret_cast<const v4f*>(parts + e);
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            const v4f x = *reinterpret_cast<const v4f*>(parts + w * BLOCK + e);
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += x[c];
        }
        const int m = m0 + e / (16 * NB), n = n0 + e % (16 * NB);
        if (m >= g.M) break;
        const int64_t at = blockIdx.z * g.bsc + m * g.ldc + n;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (n + c >= g.N) break;
            if (g.wide) static_cast<float*>(g.C)[at + c] = sum[c];
            else static_cast<uint16_t*>(g.C)[at + c] = (uint16_t)f32_to_bf16_bits(sum[c]);
        }
    }
#else
    (void)products;
#endif
}

// the workgroups of each product, and all of them
template <class Blocks>
int64_t share_out(Gemms& all, const Blocks& blocks) {
    int64_t total = 0;
    for (int i = 0; i <= TOGETHER; ++i) {
        all.first[i] = (int)total;
        if (i < all.count) total += (blocks(all.g[i]) + 7) / 8 * 8;
        if (total > 0x3fffffff) return -1;
    }
    return all.count > 1 ? total : blocks(all.g[0]);
}

template <int MB, int NB, int NW>
int launch_few(const char* fn, Gemms all, int64_t batch, hipStream_t st) {
    constexpr int LDS = MB * NB * 1024 * NW;
    static_assert(LDS <= 64 * 1024, "no limit to raise");
    int most = 0;
    for (int i = 0; i < all.count; ++i) most = all.g[i].M > most ? all.g[i].M : most;
    const int64_t strips = share_out(all, [](const Gemm& g) { return (int64_t)(g.N + 16 * NB - 1) / (16 * NB); });
    if (!idx::grid_fits(strips, 64 * NW)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    const dim3 grid((unsigned)strips, (unsigned)((most + 16 * MB - 1) / (16 * MB)), (unsigned)batch), block(64 * NW);
    if (all.count > 1)
        few_rows_kernel<MB, NB, NW, Gemms><<<grid, block, LDS, st>>>(all);
    else
        few_rows_kernel<MB, NB, NW, Gemm><<<grid, block, LDS, st>>>(all.g[0]);
    return check_launch(fn);
}

template <int BM, int BN, int WM, int WN, int STAGES>
int prepare(const char* fn, bool many) {
    constexpr int LDS = gemm_lds(BM, BN, STAGES);
    static_assert(LDS <= 160 * 1024, "LDS of a CU");
    static OncePerDevice once[2];
    const void* const kernel = many ? reinterpret_cast<const void*>(gemm_kernel<BM, BN, WM, WN, STAGES, Gemms>) : reinterpret_cast<const void*>(gemm_kernel<BM, BN, WM, WN, STAGES, Gemm>);
    if (LDS > 65536 && raise_lds_limit(once[many], kernel, LDS) != hipSuccess) return fail(TI8_ERR_HIP, "%s: %d bytes of LDS refused", fn, LDS);
    return TI8_OK;
}

template <int BM, int BN, int WM, int WN, int STAGES>
int launch(const char* fn, Gemms all, int64_t batch, hipStream_t st) {
    const int64_t tiles = share_out(all, [](Gemm& g) {
        g.tiles_m = (g.M + BM - 1) / BM;
        g.tiles_n = (g.N + BN - 1) / BN;
        return (int64_t)g.tiles_m * g.tiles_n;
    });
    if (!idx::grid_fits(tiles, 64 * WM * WN)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    if (int e = prepare<BM, BN, WM, WN, STAGES>(fn, all.count > 1)) return e;
    const dim3 grid((unsigned)tiles, (unsigned)all.g[0].parts, (unsigned)batch), block(64 * WM * WN);
    if (all.count > 1)
        gemm_kernel<BM, BN, WM, WN, STAGES, Gemms><<<grid, block, gemm_lds(BM, BN, STAGES), st>>>(all);
    else
        gemm_kernel<BM, BN, WM, WN, STAGES, Gemm><<<grid, block, gemm_lds(BM, BN, STAGES), st>>>(all.g[0]);
    return check_launch(fn);
}

// The parts of a contraction added up in order: [parts][batch][M][N] in fp32 -> C
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ from, int parts, int64_t part, int64_t rows, int M, int N, void* C, int64_t ldc, int64_t bsc, int wide) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int64_t quads = (N + 3) >> 2, at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / quads;
    if (row >= rows) return;
    const int n = (int)(at - row * quads) * 4, left = N - n;
    typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* p = from + row * N + n;
    for (int s = 0; s < parts; ++s, p += part) {
        v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (left >= 4) {
            x = *reinterpret_cast<const v4f_any*>(p);
        } else {
            for (int c = 0; c < left; ++c) x[c] = p[c];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += x[c];
    }
    const int64_t to = row / M * bsc + row % M * ldc + n;
    for (int c = 0; c < 4 && c < left; ++c) {
        if (wide) static_cast<float*>(C)[to + c] = sum[c];
        else static_cast<uint16_t*>(C)[to + c] = (uint16_t)f32_to_bf16_bits(sum[c]);
    }
#else
    (void)from; (void)parts; (void)part; (void)rows; (void)M; (void)N; (void)C; (void)ldc; (void)bsc; (void)wide;
#endif
}

}  // namespace
}  // namespace mx4
}  // namespace ti8

using namespace ti8;

namespace ti8 {
namespace mx4 {
namespace {
int launch_plan(const char* fn, int kernel, const Gemms& all, int64_t batch, hipStream_t st) {
    switch (kernel) {
        case idx::MX4_FEW_16: return launch_few<1, 1, 8>(fn, all, batch, st);
        case idx::MX4_FEW_32: return launch_few<2, 1, 8>(fn, all, batch, st);
        case idx::MX4_TILES_32: return launch<32, 64, 1, 2, 4>(fn, all, batch, st);
        case idx::MX4_TILES_64: return launch<64, 64, 2, 2, 4>(fn, all, batch, st);
        case idx::MX4_TILES_64_128: return launch<64, 128, 2, 2, 4>(fn, all, batch, st);
        case idx::MX4_TILES_128: return launch<128, 128, 2, 2, 3>(fn, all, batch, st);
        case idx::MX4_TILES_128_TWO: return launch<128, 128, 2, 2, 2>(fn, all, batch, st);
        default: return launch<256, 256, 2, 4, 2>(fn, all, batch, st);
    }
}

int64_t parts_bytes(const idx::Mx4Plan& plan, int64_t elements) { return plan.parts > 1 ? plan.parts * elements * 4 : 0; }

// What is checked of a product, and its description
int describe(const char* fn, const ti8_mx4* a, int64_t rows_a, const ti8_mx4* b, int64_t rows_b, void* c, int64_t ldc, int64_t bsc, int64_t batch, int64_t M, int64_t N,
             int64_t K, int wide, Gemm& g) {
    if (!c) return fail(TI8_ERR_NULL, "%s: a, b and c are required", fn);
    if (M <= 0 || N <= 0 || K <= 0 || batch <= 0 || batch > 65535 || M > (1 << 28) || N > (1 << 28) || K > (1 << 22) || ldc < N || bsc < 0 || (rows_a != 0 && rows_a < M) ||
        (rows_b != 0 && rows_b < N))
        return fail(TI8_ERR_SHAPE, "%s: need M, N in 1 .. 2^28, K in 1 .. 2^22, batch in 1 .. 65535, ldc >= N and batches of as many rows; got M=%lld N=%lld K=%lld batch=%lld ldc=%lld "
                    "rows_a=%lld rows_b=%lld", fn, (long long)M, (long long)N, (long long)K, (long long)batch, (long long)ldc, (long long)rows_a, (long long)rows_b);
    // (the last row that any batch reads)
    Tensor ta, tb;
    if (int e = check(fn, "a", a, (batch - 1) * rows_a + M, K, ta)) return e;
    if (int e = check(fn, "b", b, (batch - 1) * rows_b + N, K, tb)) return e;
    if (ta.ld > (1 << 22) || tb.ld > (1 << 22)) return fail(TI8_ERR_SHAPE, "%s: rows of codes may be up to 2^22 bytes apart", fn);
    if (reinterpret_cast<uintptr_t>(c) & (wide ? 3 : 1)) return fail(TI8_ERR_ALIGN, "%s: c must be aligned to its elements", fn);
    g = Gemm{ta.codes, tb.codes, ta.scales, tb.scales, c, ta.ld, tb.ld, ta.scale_ld, tb.scale_ld, rows_a, rows_b, ldc, bsc, (int)M, (int)N, (int)idx::mx4_tiles(K), 0, 0, wide ? 1 : 0, 1, 0};
    return TI8_OK;
}
}  // namespace

int init() {
    const char* const fn = "ti8_init";
    for (const bool many : {false, true}) {
        int e = prepare<32, 64, 1, 2, 4>(fn, many);
        if (!e) e = prepare<64, 64, 2, 2, 4>(fn, many);
        if (!e) e = prepare<64, 128, 2, 2, 4>(fn, many);
        if (!e) e = prepare<128, 128, 2, 2, 3>(fn, many);
        if (!e) e = prepare<128, 128, 2, 2, 2>(fn, many);
        if (!e) e = prepare<256, 256, 2, 4, 2>(fn, many);
        if (e) return e;
    }
    return TI8_OK;
}
}  // namespace mx4
}  // namespace ti8

extern "C" int64_t ti8_mx4_gemm_nt_workspace(int64_t batch, int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || batch <= 0 || batch > 65535 || M > (1 << 28) || N > (1 << 28) || K > (1 << 22)) return -1;
    return mx4::parts_bytes(idx::mx4_plan(M, N, idx::mx4_tiles(K), batch, device_cu_count()), batch * M * N);
}

extern "C" int ti8_mx4_gemm_nt(const ti8_mx4* a, int64_t rows_a, const ti8_mx4* b, int64_t rows_b, void* c, int64_t ldc, int64_t bsc, int64_t batch, int64_t M, int64_t N,
                               int64_t K, int wide, void* workspace, int64_t workspace_bytes, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_gemm_nt";
    if (!a || !b) return fail(TI8_ERR_NULL, "%s: a, b and c are required", fn);
    mx4::Gemms all;
    all.count = 1;
    mx4::Gemm& g = all.g[0];
    if (int e = mx4::describe(fn, a, rows_a, b, rows_b, c, ldc, bsc, batch, M, N, K, wide, g)) return e;
    const idx::Mx4Plan plan = idx::mx4_plan(M, N, g.nk, batch, device_cu_count());
    const int64_t need = mx4::parts_bytes(plan, batch * M * N);
    if (need && (!workspace || workspace_bytes < need)) return fail(TI8_ERR_NULL, "%s: a workspace of %lld bytes is required", fn, (long long)need);
    if (need && !aligned16(workspace)) return fail(TI8_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", fn);
    if (need) {
        g.C = workspace;
        g.wide = 1;
        g.ldc = N;
        g.bsc = M * N;
        g.parts = plan.parts;
        g.part = batch * M * N;
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = need ? (batch * M * ((N + 3) / 4) + 255) / 256 : 0;
    if (need && !idx::grid_fits(blocks, 256)) return fail(TI8_ERR_SHAPE, "%s: too many elements for one call", fn);
    if (int e = mx4::launch_plan(fn, plan.kernel, all, batch, st)) return e;
    if (!need) return TI8_OK;
    mx4::join_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(static_cast<const float*>(workspace), plan.parts, g.part, batch * M, (int)M, (int)N, c, ldc, bsc, wide ? 1 : 0);
    return check_launch(fn);
}

extern "C" int64_t ti8_mx4_gemm_nt_multi_workspace(const ti8_mx4_gemm_problem* problems, int count) {
    if (!problems || count < 1 || count > mx4::TOGETHER) return -1;
    int64_t sizes[mx4::TOGETHER][3], most = 0;
    for (int i = 0; i < count; ++i) {
        const ti8_mx4_gemm_problem& p = problems[i];
        const int64_t need = ti8_mx4_gemm_nt_workspace(1, p.M, p.N, p.K);
        if (need < 0) return -1;
        if (need > most) most = need;
        sizes[i][0] = p.M;
        sizes[i][1] = p.N;
        sizes[i][2] = idx::mx4_tiles(p.K);
    }
    return count > 1 && idx::mx4_plan_together(sizes, count, device_cu_count()) >= 0 ? 0 : most;
}

extern "C" int ti8_mx4_gemm_nt_multi(const ti8_mx4_gemm_problem* problems, int count, void* workspace, int64_t workspace_bytes, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_gemm_nt_multi";
    if (!problems) return fail(TI8_ERR_NULL, "%s: problems are required", fn);
    if (count < 1 || count > mx4::TOGETHER) return fail(TI8_ERR_SHAPE, "%s: need 1 to %d products, got %d", fn, mx4::TOGETHER, count);
    mx4::Gemms all;
    all.count = count;
    int64_t sizes[mx4::TOGETHER][3];
    // the longest contractions first: the short ones fill up what they leave
    int order[mx4::TOGETHER] = {0, 1, 2};
    for (int i = 1; i < count; ++i)
        for (int j = i; j > 0 && problems[order[j]].K > problems[order[j - 1]].K; --j) {
            const int t = order[j];
            order[j] = order[j - 1];
            order[j - 1] = t;
        }
    for (int i = 0; i < count; ++i) {
        const ti8_mx4_gemm_problem& p = problems[order[i]];
        if (int e = mx4::describe(fn, &p.a, 0, &p.b, 0, p.c, p.ldc, 0, 1, p.M, p.N, p.K, p.wide, all.g[i])) return e;
        int64_t* const size = sizes[order[i]];     // (in the caller's order, as the workspace was asked for: the plan's sums are the same)
        size[0] = p.M;
        size[1] = p.N;
        size[2] = all.g[i].nk;
    }
    const int kernel = count > 1 ? idx::mx4_plan_together(sizes, count, device_cu_count()) : -1;
    if (kernel >= 0) return mx4::launch_plan(fn, kernel, all, 1, static_cast<hipStream_t>(stream));
    const int64_t need = ti8_mx4_gemm_nt_multi_workspace(problems, count);
    if (need && (!workspace || workspace_bytes < need)) return fail(TI8_ERR_NULL, "%s: a workspace of %lld bytes is required", fn, (long long)need);
    if (need && !aligned16(workspace)) return fail(TI8_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", fn);
    for (int i = 0; i < count; ++i) {
        const ti8_mx4_gemm_problem& p = problems[i];
        if (int e = ti8_mx4_gemm_nt(&p.a, 0, &p.b, 0, p.c, p.ldc, 0, 1, p.M, p.N, p.K, p.wide, workspace, workspace_bytes, stream)) return e;
    }
    return TI8_OK;
}

namespace {
// Where a step's operands lie in its workspace: X, W and dY by rows and by columns, and behind them what the products need
struct Mx4Step {
    ti8_mx4_operand o[3];
    ti8_mx4_gemm_problem p[3];
    int64_t products, bytes;
    bool ok;
};
Mx4Step mx4_step(int64_t T, int64_t K, int64_t N, char* base) {
    Mx4Step s{};
    s.ok = T > 0 && K > 0 && N > 0 && T <= (1 << 22) && K <= (1 << 22) && N <= (1 << 22);
    if (!s.ok) return s;
    const auto take = [&](int64_t bytes) {
        char* const at = base + s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    const auto room = [&](int64_t rows, int64_t cols) {
        const int64_t tiles = idx::mx4_tiles(cols);
        ti8_mx4 t;
        t.ld = tiles * idx::MX4_TILE_BYTES;
        t.scale_ld = rows * idx::MX4_TILE_SCALES;
        t.codes = take(rows * t.ld);
        t.scales = take(tiles * t.scale_ld);
        return t;
    };
    const int64_t rows[3] = {T, N, T}, cols[3] = {K, K, N};
    for (int i = 0; i < 3; ++i) {
        s.o[i].rows = rows[i];
        s.o[i].cols = cols[i];
        s.o[i].by_rows = room(rows[i], cols[i]);
        s.o[i].by_columns = room(cols[i], rows[i]);
    }
    const ti8_mx4_operand &x = s.o[0], &w = s.o[1], &d = s.o[2];
    s.p[0] = {x.by_rows, w.by_rows, nullptr, N, T, N, K, 0};
    s.p[1] = {d.by_rows, w.by_columns, nullptr, K, T, K, N, 0};
    s.p[2] = {d.by_columns, x.by_columns, nullptr, K, N, K, T, 0};
    s.products = ti8_mx4_gemm_nt_multi_workspace(s.p, 3);
    take(s.products);
    return s;
}
}  // namespace

extern "C" int64_t ti8_mx4_linear_fwd_bwd_workspace(int64_t T, int64_t K, int64_t N) {
    const Mx4Step s = mx4_step(T, K, N, nullptr);
    return s.ok ? s.bytes : -1;
}

extern "C" int ti8_mx4_linear_fwd_bwd(const void* X, int64_t ldx, const void* W, int64_t ldw, const void* dY, int64_t lddy, void* Y, void* dX, void* dW,
                                      int64_t T, int64_t K, int64_t N, void* workspace, int64_t workspace_bytes, ti8_stream_t stream) {
    const char* const fn = "ti8_mx4_linear_fwd_bwd";
    if (!X || !W || !dY || !Y || !dX || !dW || !workspace) return fail(TI8_ERR_NULL, "%s: X, W, dY, Y, dX, dW and workspace are required", fn);
    Mx4Step s = mx4_step(T, K, N, static_cast<char*>(workspace));
    if (!s.ok) return fail(TI8_ERR_SHAPE, "%s: need T, K, N in 1 .. 2^22; got T=%lld K=%lld N=%lld", fn, (long long)T, (long long)K, (long long)N);
    if (workspace_bytes < s.bytes) return fail(TI8_ERR_NULL, "%s: a workspace of %lld bytes is required, got %lld", fn, (long long)s.bytes, (long long)workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) || ((reinterpret_cast<uintptr_t>(Y) | reinterpret_cast<uintptr_t>(dX) | reinterpret_cast<uintptr_t>(dW)) & 1))
        return fail(TI8_ERR_ALIGN, "%s: the workspace must be 256-byte aligned, outputs 2-byte", fn);
    const void* const x[3] = {X, W, dY};
    const int64_t ld[3] = {ldx, ldw, lddy};
    for (int i = 0; i < 3; ++i) {
        s.o[i].x = x[i];
        s.o[i].ldx = ld[i];
    }
    // (from here on everything is checked that the calls below check, but for the inputs' leading dimensions and alignment, which the first of them checks before it
    // launches anything)
    if (int e = ti8_mx4_quant(s.o, 3, stream)) return e;
    char* const products = static_cast<char*>(workspace) + (s.bytes - (s.products + 255) / 256 * 256);
    void* const to[3] = {Y, dX, dW};
    for (int i = 0; i < 3; ++i) s.p[i].c = to[i];
    return ti8_mx4_gemm_nt_multi(s.p, 3, products, s.products, stream);
}
