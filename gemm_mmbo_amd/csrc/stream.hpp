// A few columns against weights that are read once: a wavefront streams rows of weights past up to 32 columns.
//
// D(column, row) += X(column, l) * W(l, row) on 16x16x32 MFMAs, weights as the second operand: lane l holds row l % 16, eight places of k from
// 8 * (l / 16) on, and of the results row l % 16 for columns 4 * (l / 16) .. + 3.  A row's scale and zero point are then those of the lane.
// Each wavefront of a work-group has the same rows and a run of k of its own; the sums meet in LDS at the end, in the order of the wavefronts.
//
// Weights, their scales and columns go through a ring of the wavefront's own in LDS that direct loads fill, DEPTH blocks ahead: no barrier before the sums,
// no register for what is under way.  Loads have to come as whole memory lines: with a lane to a row, as MFMAs want them, a CU got 11 bytes a clock
// (4096 x 16 x 14336 in 4 bits: 24 us), with 64 bytes to four lanes 20 (13.3 us), though halves of a line were asked for one behind the other.
//
// 4-bit weights: a block is 128 places, half a line of a row (whole lines took a sixth longer with one column: 33 us for 28, before scales went through the ring).  Eight codes become numbers by moving nibbles to where a mantissa ends:
//   fp16: a subnormal number, code * 2^-24, of which a packed fma makes (code - zero) * 2^-10: 11 instructions.  Not the subnormal numbers themselves: an MFMA lines its
//     products up by the operands' exponents, which are then 10 to 13 above the products, and cuts off what fp32 would hold (one in twenty of a product's results was another fp16 number).
//   bf16: a byte of 0 .. 15 is that many 2^-9 in e4m3, of which the conversion with a scale makes the code, exact: 9 instructions.  A second MFMA behind each one
//     takes zero * column off, 32 places at a time.  Not 128 + code and zero + 128 off the group's sums: those take bits from what is left.  Or (LESS_ZERO) from the
//     subnormal fp16 number one mixed-precision fma makes code - zero in fp32, and two of those are packed: 19 instructions and no second MFMA (28672 x 1 x 8192 38.0 us
//     for 34.7, 8192 x 1 x 8192 11.5 for 10.0).
// A group's sums are multiplied by its scale, in fp32.
// 16-bit weights: a block is 64 places, a line of a row.
//
// What bounds it: one column, the weights from memory beside requests of scales, a line a row and block (28672 x 1 x 8192: 31.6 us in either type, with zero points 34.7, for
// 119 and 121 MB, which take 21; 4096 x 1 x 4096 5.0 us, a launch).  More columns, what a CU gets from the L2, some 50 bytes a ns: each work-group reads all columns for its 16
// or 32 rows (4096 x 16 x 14336 12.9 us for 0.6 MB a CU, 8192 x 64 x 8192 26.5 for 1.3 MB).
#pragma once

#include <type_traits>

#include "gemm_ring.hpp"
#include "w4.hpp"

namespace mmbo {

namespace stream {

typedef u32x4 __attribute__((aligned(1))) u32x4_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Type;
template <> struct Type<half_t> {
    typedef f16x8 Frag;
    __device__ static inline f32x4 mfma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Type<bf16_t> {
    typedef bf16x8 Frag;
    __device__ static inline f32x4 mfma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template <typename T>
__device__ inline typename Type<T>::Frag frag_of(u32x4 v)
{
    return __builtin_bit_cast(typename Type<T>::Frag, v);
}

// Eight elements from `p`, of which `here` exist (any number; none: no access); the others are 0.
template <typename T>
__device__ inline u32x4 load8(const T *p, int64_t here)
{
    if (here >= 8) return *reinterpret_cast<const u32x4_any *>(p);
    union { uint16_t e[8]; u32x4 v; } u;
    u.v = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < here) u.e[i] = __builtin_bit_cast(uint16_t, p[i]);
    return u.v;
}
// 32 codes from `p`, of which `here` exist; the others may be anything.
__device__ inline u32x4 load32_codes(const uint8_t *p, int64_t here)
{
    union { uint8_t e[16]; u32x4 v; } u;
    u.v = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (2 * i < here) u.e[i] = p[i];
    return u.v;
}

// Eight numbers from a dword of codes, exact: kUnit times the code, less the zero point (always with LESS_ZERO) or not.
template <typename T, bool LESS_ZERO = false> struct Codes;
template <bool LESS_ZERO> struct Codes<half_t, LESS_ZERO> {
    static constexpr bool kLessZero = true;
    static constexpr float kUnit = 0x1p-10f;
    typedef f16x2 Zero;
    __device__ static inline Zero zero_of(uint32_t z)
    {
        const half_t v = (half_t)((float)z * -kUnit);
        return Zero{v, v};
    }
    __device__ static inline f16x8 expand(uint32_t x, const Zero &z)
    {
        union { f16x2 h[4]; f16x8 v; } u;
        const uint32_t even = x & 0x0F0F0F0Fu, odd = x >> 4 & 0x0F0F0F0Fu;
        const f16x2 up = {(half_t)0x1p14f, (half_t)0x1p14f};
#pragma unroll
        for (int p = 0; p < 4; ++p)                     // byte p of either
            u.h[p] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(odd, even, 0x0c040c00u + p * 0x00010001u)), up, z);
        return u.v;
    }
};
template <> struct Codes<bf16_t, false> {
    static constexpr bool kLessZero = false;
    static constexpr float kUnit = 1.0f;
    typedef bf16x8 Zero;                                // what comes off, as a second operand
    __device__ static inline Zero zero_of(uint32_t z)
    {
        const bf16_t v = (bf16_t)-(float)z;
        return Zero{v, v, v, v, v, v, v, v};
    }
    __device__ static inline bf16x8 expand(uint32_t x, const Zero &)
    {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        union { bf16x2 h[4]; bf16x8 v; } u;
        const uint32_t even = x & 0x0F0F0F0Fu, odd = x >> 4 & 0x0F0F0F0Fu;
        const uint32_t low = __builtin_amdgcn_perm(odd, even, 0x05010400u), high = __builtin_amdgcn_perm(odd, even, 0x07030602u);   // codes 0 .. 3, 4 .. 7
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 0x1p9f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 0x1p9f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 0x1p9f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 0x1p9f, true);
        return u.v;
    }
};

template <> struct Codes<bf16_t, true> {
    static constexpr bool kLessZero = true;
    static constexpr float kUnit = 1.0f;
    typedef float Zero;
    __device__ static inline Zero zero_of(uint32_t z) { return -(float)z; }
    __device__ static inline bf16x8 expand(uint32_t x, Zero z)
    {
        bf16x8 v;
        const uint32_t even = x & 0x0F0F0F0Fu, odd = x >> 4 & 0x0F0F0F0Fu;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(odd, even, 0x0c040c00u + p * 0x00010001u));
            v[2 * p] = (bf16_t)__builtin_fmaf((float)h[0], 0x1p24f, z);
            v[2 * p + 1] = (bf16_t)__builtin_fmaf((float)h[1], 0x1p24f, z);
        }
        return v;
    }
};

// 16 bytes a lane from `p` to LDS at lds_addr + 16 * lane; 2 bytes or 1, as a dword, to lds_addr + 4 * lane (lanes that take no part leave theirs as it
// is).  As ring::direct_load16, but from an address a lane: rows may lie anywhere.  (The instruction's offset counts for both places.)
template <int OFFSET = 0>
__device__ inline void direct_load(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%2" ::"v"(p), "s"(lds_addr - OFFSET), "n"(OFFSET) : "memory");
}
__device__ inline void direct_load_u16(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ushort %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}
__device__ inline void direct_load_u8(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}

// Rows of 128 bytes in LDS as direct loads put them: lane l loads a 16-byte chunk of row l / 8 (of eight, and of the eight behind them with the next load), and the
// place that is its own takes chunk (l % 8) ^ (row / 2 % 8).  The exclusive or spreads over the banks what is read together: one chunk of 16 rows, or a dword of
// each of four lanes' chunks.  Rows of 64 bytes: row l / 4, chunk (l % 4) ^ (row / 4 % 4).
template <int ROW_BYTES>
__device__ inline uint32_t chunk_of(uint32_t row, int lane) { return ROW_BYTES == 64 ? (lane & 3) ^ (row >> 2 & 3) : (lane & 7) ^ (row >> 1 & 7); }
template <int ROW_BYTES>
__device__ inline uint32_t chunk_at(uint32_t row, uint32_t chunk)
{
    return ROW_BYTES == 64 ? row * 64 + ((chunk ^ (row >> 2 & 3)) << 4) : row * 128 + ((chunk ^ (row >> 1 & 7)) << 4);
}

// The sums of a wavefront over its share of several jobs: of each job blocks block0 .. block0 + per_job - 1 of k, job after job, and of all these blocks
// numbers first .. first + count - 1.  enter(job, Job &) says where its operands lie, flush(job, sums) takes the sums of what the wavefront had of it.  Results
// of columns that do not exist are not defined.  lds: the wavefront's own LDS_BYTES.
// T: of weights and scales; TX: of the columns, and what is multiplied -- with TX bf16, T may be fp16.
// N2: columns side by side, 1, 4, 16 or 32, each in PLANES numbers of type TX, which are added.  FT: tiles of 16 rows.  LESS_ZERO: of Codes.
// FP32: columns in fp32 in the room of two planes, four places of eight in each; the last eight are whole ones.
// FOLD (4-bit weights): places whose sums are multiplied by a scale at once: 128 where groups are whole multiples of that, 64, else 32.
template <typename T, bool W4, int N2, int FT, int PLANES, int FOLD, bool ZEROS, int DEPTH, typename TX = T, bool LESS_ZERO = false, bool FP32 = false>
struct Stream {
    static_assert(N2 == 1 || N2 == 4 || N2 == 16 || N2 == 32, "");
    typedef typename Type<TX>::Frag Frag;
    typedef typename Codes<TX, LESS_ZERO>::Zero Zero;
    static constexpr int NT = N2 > 16 ? N2 / 16 : 1, BLOCK = W4 ? 128 : 64, STEPS = BLOCK / 32, ROW_BYTES = W4 ? BLOCK / 2 : 128;
    static constexpr int FOLDS = W4 ? BLOCK / FOLD : 1;
    static constexpr int WP = ROW_BYTES / 64, W_TILE = WP * 1024;
    static constexpr int X_LINES = BLOCK / 64, XP = N2 < 8 ? 1 : N2 / 8, X_LANES = X_LINES * N2 * 8 < 64 ? X_LINES * N2 * 8 : 64,
                         X_LOADS = (X_LINES * N2 * 8 + 63) / 64, X_PLANE = X_LINES * N2 * 128;
    static constexpr int S_LOADS = W4 ? (FOLDS + 3) / 4 : 0, S_TILE = FOLDS * 64;
    static constexpr int X_AT = FT * W_TILE, S_AT = X_AT + PLANES * X_PLANE, Z_AT = S_AT + (W4 ? FT * S_TILE : 0), SLOT = (Z_AT + (W4 && ZEROS ? FT * S_TILE : 0) + 127) / 128 * 128;
    static constexpr bool S_ONE = W4 && FT * FOLDS <= 4;          // one load has the scales of all tiles (8192 x 16 x 8192 11.5 us, with one a tile 12.2)
    static constexpr int LOADS = FT * WP + PLANES * X_LOADS + (S_ONE ? 1 : FT * S_LOADS) * (ZEROS ? 2 : 1);
    static constexpr int LDS_BYTES = (DEPTH * SLOT + 1023) / 1024 * 1024;
    static_assert((DEPTH - 1) * LOADS < 64, "vmcnt counts to 63");
    typedef f32x4 Sums[NT][FT];
    // A wavefront's sums in LDS: of a tile all columns that there may be.
    static constexpr int TILE_FLOATS = N2 < 16 ? 16 * N2 : 256, SET_FLOATS = NT * FT * TILE_FLOATS;
    __device__ static inline void put(float *to, const Sums &acc, int lane)
    {
        if (N2 < 16 && lane >= 16) return;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int f = 0; f < FT; ++f) {
                if constexpr (N2 == 1) to[(c * FT + f) * TILE_FLOATS + lane] = acc[c][f][0];
                else *reinterpret_cast<f32x4 *>(to + (c * FT + f) * TILE_FLOATS + lane * 4) = acc[c][f];
            }
    }
    // What `waves` wavefronts have of row `row` of tile f and column `col`, added in their order; set: the first one's.
    __device__ static inline float total(const float *set, uint32_t f, uint32_t row, uint32_t col, uint32_t waves)
    {
        const float *at = set + (col / 16 * FT + f) * TILE_FLOATS + (N2 == 1 ? row : ((col >> 2 & 3) * 16 + row) * 4 + (col & 3));
        float v = at[0];
        for (uint32_t w = 1; w < waves; ++w) v += at[w * SET_FLOATS];
        return v;
    }
    // Every wavefront of the work-group has put its sums (not __syncthreads(): what is under way stays so).
    __device__ static inline void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

    // Where a lane finds a job's rows of weights and its columns, from their first place on.  In the place of those that do not exist: others that do.
    struct Job {
        const uint8_t *w[FT][WP];               // rows load_row(lane, 0 ..) of a tile: of codes, or of elements
        const T *scales[FT];                    // row lane % 16
        const uint8_t *zeros[FT];
        const TX *x[PLANES][XP];                 // columns load_column(lane, 0 ..)
        bool x_here[XP];                        // .. exist
    };
    __device__ static inline uint32_t load_row(int lane, int p) { return ROW_BYTES == 64 ? lane >> 2 : p * 8 + (lane >> 3); }
    __device__ static inline uint32_t load_column(int lane, int p) { return N2 < 8 ? (lane >> 3) & (N2 - 1) : p * 8 + (lane >> 3); }
    // of load j: the first place of its line in the block
    __device__ static inline uint32_t x_line(int lane, int j) { return 64 * (N2 < 8 ? lane / (8 * N2) + j * (8 / N2) : j / XP); }
    __device__ static inline uint32_t w_chunk(int lane, int p) { return chunk_of<ROW_BYTES>(load_row(lane, p), lane); }
    __device__ static inline uint32_t x_chunk(int lane, int p) { return chunk_of<128>(load_column(lane, p), lane); }
    __host__ __device__ static inline uint32_t blocks_of(uint32_t k) { return (k + BLOCK - 1) / BLOCK; }

    uint32_t k, group32;                        // places; places of a group / 32
    char *lds;
    int lane;
    uint32_t lds_at, block0, per_job;
    // requests
    Job from;
    uint32_t r_job, r_block, group[S_LOADS + 1], rest[S_LOADS + 1];                     // (of the lane's folds)
    // products
    struct Operands {
        Frag x[PLANES][STEPS][NT];
        u32x4 w[W4 ? 1 : STEPS][FT];
        uint32_t codes[W4 ? STEPS : 1][FT];
        uint32_t scales[FOLDS][FT], zeros[FOLDS][FT];
    } o;

    __device__ inline Stream(uint32_t k, uint32_t group32, uint32_t block0, uint32_t per_job, char *lds, int lane)
        : k(k), group32(group32), lds(lds), lane(lane), lds_at(__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MMBO_LDS_PTR(lds))), block0(block0),
          per_job(per_job)
    {
    }

    template <typename Enter>
    __device__ inline void enter_job(const Enter &enter)
    {
        enter(r_job, from);
        const uint32_t b = block0 + r_block;
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int p = 0; p < WP; ++p) from.w[f][p] += (uint64_t)b * ROW_BYTES + w_chunk(lane, p) * 16;
#pragma unroll
        for (int p = 0; p < XP; ++p) {
            // (a load without a lane is none, and would not count: the first column of an eight comes in any case)
            from.x_here[p] = (from.x_here[p] || lane < 8) && lane < X_LANES;
#pragma unroll
            for (int q = 0; q < PLANES; ++q) from.x[q][p] += b * BLOCK + x_chunk(lane, p) * 8 + (N2 < 8 ? x_line(lane, 0) : 0);
        }
        if constexpr (S_ONE && FT == 2)
            if (lane >= 16 * FOLDS) {
                from.scales[0] = from.scales[1];
                if constexpr (ZEROS) from.zeros[0] = from.zeros[1];
            }
#pragma unroll
        for (int j = 0; j < S_LOADS; ++j) {
            const uint32_t at = b * STEPS + (S_ONE ? (lane >> 4) % FOLDS : j * 4 + (lane >> 4)) * (STEPS / FOLDS);
            group[j] = at / group32;
            rest[j] = at % group32;
        }
    }
    template <typename Enter>
    __device__ inline void request(uint32_t slot, const Enter &enter)
    {
        if (r_block == per_job) {
            ++r_job;
            r_block = 0;
            enter_job(enter);
        }
        const uint32_t to = lds_at + slot * SLOT;
        // scales: lane's row lane % 16, its folds lane / 16 and every fourth behind that; or in one load tile lane / (16 * FOLDS), fold lane / 16 % FOLDS
#pragma unroll
        for (int j = 0; j < S_LOADS; ++j) {
            const uint32_t g = min(group[j], (k - 1) / 32 / group32);
            if (lane < 16 * FOLDS * (S_ONE ? FT : 1) || FOLDS >= 4)
#pragma unroll
                for (int f = 0; f < (S_ONE ? 1 : FT); ++f) {
                    direct_load_u16(from.scales[f] + g, to + S_AT + f * S_TILE + j * 256);
                    if constexpr (ZEROS) direct_load_u8(from.zeros[f] + g, to + Z_AT + f * S_TILE + j * 256);
                }
            group[j] += STEPS / group32;
            rest[j] += STEPS % group32;
            if (rest[j] >= group32) { rest[j] -= group32; ++group[j]; }
        }
        if ((block0 + r_block) * BLOCK + BLOCK <= k) {
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int p = 0; p < WP; ++p) direct_load(from.w[f][p], to + f * W_TILE + p * 1024);
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
                ring::static_for<X_LOADS>([&](auto J) {
                    constexpr int j = decltype(J)::value;
                    if (from.x_here[j % XP]) direct_load<(N2 < 8 ? j * (8 / N2) : j / XP) * 128>(from.x[q][j % XP], to + X_AT + q * X_PLANE + j * 1024);
                });
        } else {
            // The last block of a k that is not a whole number of them, through registers.  Counts of what is under way no longer hold then, so nothing is,
            // for once.
            const int64_t left = (int64_t)k - (block0 + r_block) * BLOCK;
            char *const slot_at = lds + slot * SLOT;
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int p = 0; p < WP; ++p) {
                    const int64_t here = left - w_chunk(lane, p) * (W4 ? 32 : 8);
                    u32x4 *const at = reinterpret_cast<u32x4 *>(slot_at + f * W_TILE + p * 1024 + lane * 16);
                    if constexpr (W4) *at = here >= 32 ? *reinterpret_cast<const u32x4_any *>(from.w[f][p]) : load32_codes(from.w[f][p], here);
                    else *at = load8(reinterpret_cast<const T *>(from.w[f][p]), here);
                }
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
#pragma unroll
                for (int j = 0; j < X_LOADS; ++j)
                    if (from.x_here[j % XP]) {
                        const int64_t here = (left - x_line(lane, j) - x_chunk(lane, j % XP) * 8 + (FP32 ? 7 : 0)) & (FP32 ? ~7 : ~0);
                        *reinterpret_cast<u32x4 *>(slot_at + X_AT + q * X_PLANE + j * 1024 + lane * 16) = load8(from.x[q][j % XP] + x_line(0, j), here);
                    }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        ++r_block;
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int p = 0; p < WP; ++p) from.w[f][p] += ROW_BYTES;
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
#pragma unroll
            for (int p = 0; p < XP; ++p) from.x[q][p] += BLOCK;
    }

    __device__ inline void read(uint32_t slot)
    {
        const uint32_t row = lane & 15, quarter = lane >> 4;
        const char *const at = lds + slot * SLOT;
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int c = 0; c < NT; ++c)
                    o.x[q][i][c] = frag_of<TX>(*reinterpret_cast<const u32x4 *>(at + X_AT + q * X_PLANE + i / 2 * N2 * 128 +
                                                                               chunk_at<128>((lane & (N2 < 16 ? N2 - 1 : 15)) + c * 16, i % 2 * 4 + quarter)));
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            if constexpr (W4) {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) o.codes[i][f] = *reinterpret_cast<const uint32_t *>(at + f * W_TILE + chunk_at<ROW_BYTES>(row, i) + quarter * 4);
#pragma unroll
                for (int q = 0; q < FOLDS; ++q) {
                    o.scales[q][f] = *reinterpret_cast<const uint32_t *>(at + S_AT + f * S_TILE + (q * 16 + row) * 4);
                    if constexpr (ZEROS) o.zeros[q][f] = *reinterpret_cast<const uint32_t *>(at + Z_AT + f * S_TILE + (q * 16 + row) * 4);
                }
            } else {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) o.w[i][f] = *reinterpret_cast<const u32x4 *>(at + f * W_TILE + chunk_at<128>(row, i * 4 + quarter));
            }
        }
    }

    // What the MFMAs take of tile c of columns and 32 places: its planes, or fp32 in three bf16 numbers, cut off where one ends (finite numbers exactly).
    static constexpr int kParts = FP32 ? 3 : PLANES;
    __device__ inline void parts(Frag (&x)[kParts], int i, int c) const
    {
        if constexpr (FP32) {
            union { Frag from[2]; uint32_t u[8]; float v[8]; } h;
            h.from[0] = o.x[0][i][c];
            h.from[1] = o.x[1][i][c];
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                union { uint32_t d[4]; Frag v; } u;
#pragma unroll
                for (int p = 0; p < 4; ++p) u.d[p] = __builtin_amdgcn_perm(h.u[2 * p + 1], h.u[2 * p], 0x07060302u);
                x[e] = u.v;
                if (e < 2)
#pragma unroll
                    for (int p = 0; p < 8; ++p) h.v[p] -= __builtin_bit_cast(float, h.u[p] & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < PLANES; ++e) x[e] = o.x[e][i][c];
        }
    }
    __device__ inline void multiply(Sums &acc)
    {
        if constexpr (W4) {
#pragma unroll
            for (int q = 0; q < FOLDS; ++q) {
                Sums part;
                Zero zero[FT];
                clear(part);
#pragma unroll
                for (int f = 0; f < FT; ++f) zero[f] = Codes<TX, LESS_ZERO>::zero_of(ZEROS ? o.zeros[q][f] & kW4ZeroMask : (uint32_t)kW4Zero);
#pragma unroll
                for (int i = q * (STEPS / FOLDS); i < (q + 1) * (STEPS / FOLDS); ++i) {
                    Frag w[FT];
#pragma unroll
                    for (int f = 0; f < FT; ++f) w[f] = Codes<TX, LESS_ZERO>::expand(o.codes[i][f], zero[f]);
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                        Frag x[kParts];
                        parts(x, i, c);
#pragma unroll
                        for (int f = 0; f < FT; ++f)
#pragma unroll
                            for (int e = 0; e < kParts; ++e) {
                                part[c][f] = Type<TX>::mfma(x[e], w[f], part[c][f]);
                                if constexpr (!Codes<TX, LESS_ZERO>::kLessZero) part[c][f] = Type<TX>::mfma(x[e], zero[f], part[c][f]);
                            }
                    }
                }
#pragma unroll
                for (int f = 0; f < FT; ++f) {
                    const float s = (float)__builtin_bit_cast(T, (uint16_t)o.scales[q][f]) * (1.0f / Codes<TX, LESS_ZERO>::kUnit);
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[c][f][r] = __builtin_fmaf(s, part[c][f][r], acc[c][f][r]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    Frag x[kParts];
                    parts(x, i, c);
#pragma unroll
                    for (int f = 0; f < FT; ++f) {
                        Frag w[kWeightPlanes];
                        weights(w, o.w[i][f]);
#pragma unroll
                        for (int e = 0; e < kParts; ++e)
#pragma unroll
                            for (int p = 0; p < kWeightPlanes; ++p) acc[c][f] = Type<TX>::mfma(x[e], w[p], acc[c][f]);
                    }
                }
        }
    }
    // Weights of 16 bits as second operands: as they are, or fp16 in two bf16 numbers, 8 and 3 bits of its 11 (finite numbers exactly).
    static constexpr int kWeightPlanes = __is_same(T, TX) ? 1 : 2;
    __device__ static inline void weights(Frag (&w)[kWeightPlanes], u32x4 v)
    {
        if constexpr (kWeightPlanes == 1) {
            w[0] = frag_of<TX>(v);
        } else {
            const f16x8 high = frag_of<T>(v & 0xFFF8FFF8u), low = frag_of<T>(v) - high;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[0][i] = (TX)(float)high[i];
                w[1][i] = (TX)(float)low[i];
            }
        }
    }
    __device__ static inline void clear(Sums &acc)
    {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int f = 0; f < FT; ++f) acc[c][f] = f32x4{0, 0, 0, 0};
    }

    template <typename Enter, typename Flush>
    __device__ inline void run(uint32_t first, uint32_t count, const Enter &enter, const Flush &flush)
    {
        if (count == 0) return;
        Sums acc;
        clear(acc);
        uint32_t job = first / per_job, block = first % per_job;
        r_job = job;
        r_block = block;
        enter_job(enter);
#pragma unroll
        for (int s = 0; s < DEPTH; ++s)
            if ((uint32_t)s < count) request(s, enter);
        auto product = [&] {
            multiply(acc);
            if (++block == per_job) {
                flush(job, acc);
                clear(acc);
                ++job;
                block = 0;
            }
        };
        // (the compiler does not count direct loads; the "memory" clobbers keep what is read between them)
        uint32_t slot = 0, s = 0;
        for (; s + DEPTH < count; ++s) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * LOADS) : "memory");
            read(slot);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                   // in registers: the slot is free
            request(slot, enter);
            product();
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (; s < count; ++s) {
            read(slot);
            product();
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        if (block != 0) flush(job, acc);
    }
};

}  // namespace stream

// A unit of work: 16 * FT rows of W, N2 columns of B, k shared by the wavefronts.  A work-group takes a run of units, one behind the other without a pause in its
// loads: the wavefronts meet once a unit, over two sets of sums in turn.
template <typename T, int N2, int FT, int FOLD, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(512)
gemm_w4_stream_kernel(const GemmW4Args a)
{
    using namespace stream;
    typedef Stream<T, true, N2, FT, 1, FOLD, ZEROS, DEPTH> S;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t all = (a.m + 16 * FT - 1) / (16 * FT), col0 = blockIdx.y * N2;
    const uint32_t unit0 = (uint32_t)((uint64_t)all * blockIdx.x / gridDim.x), units = (uint32_t)((uint64_t)all * (blockIdx.x + 1) / gridDim.x) - unit0;
    float *const sums = reinterpret_cast<float *>(lds + waves * S::LDS_BYTES);           // [set][wavefront][..]
    auto enter = [&](uint32_t u, typename S::Job &j) {
        const uint32_t row0 = (unit0 + u) * 16 * FT;
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            const uint64_t i = min(row0 + f * 16 + (lane & 15), a.m - 1);               // (rows past the edge repeat the last one)
#pragma unroll
            for (int q = 0; q < S::WP; ++q) j.w[f][q] = a.w.q + (uint64_t)min(row0 + f * 16 + S::load_row(lane, q), a.m - 1) * a.w.ldq;
            j.scales[f] = static_cast<const T *>(a.w.scales) + i * a.w.lds;
            j.zeros[f] = ZEROS ? a.w.zeros + i * a.w.ldz : nullptr;
        }
#pragma unroll
        for (int q = 0; q < S::XP; ++q) {
            const uint32_t col = col0 + S::load_column(lane, q);
            j.x[0][q] = static_cast<const T *>(a.B) + min(col, a.n - 1) * a.ldb;
            j.x_here[q] = col < a.n;
        }
    };
    auto flush = [&](uint32_t u, const typename S::Sums &acc) {
        float *const set = sums + (u & 1) * waves * S::SET_FLOATS;
        S::put(set + wave * S::SET_FLOATS, acc, lane);
        S::meet();
        const uint32_t row0 = (unit0 + u) * 16 * FT;
        for (uint32_t at = threadIdx.x; at < 16 * FT * N2; at += blockDim.x) {
            const uint32_t f = at / 16 % FT, col = at / (16 * FT), i = row0 + f * 16 + (at & 15), j = col0 + col;
            if (i >= a.m || j >= a.n) continue;
            T *c = static_cast<T *>(a.C) + i + j * a.ldc;
            float v = a.alpha * S::total(set, f, at & 15, col, waves);
            if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*c, v);
            *c = (T)v;
        }
    };
    const uint32_t blocks = S::blocks_of(a.k), each = blocks / waves, more = blocks % waves, mine = each + (wave < more);
    S s(a.k, a.group / kW4Group, wave * each + min(wave, more), mine, lds + wave * S::LDS_BYTES, lane);
    if (mine != 0) {
        s.run(0, units * mine, enter, flush);
    } else {                                                                            // k is 0: nothing to add
        typename S::Sums none;
        S::clear(none);
        for (uint32_t u = 0; u < units; ++u) flush(u, none);
    }
}

}  // namespace mmbo
