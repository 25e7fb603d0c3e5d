// A few columns against weights that are read once: a wavefront streams rows of weights past up to 32 columns.
//
// D(column, row) += X(column, l) * W(l, row) on 16x16x32 MFMAs, weights as the second operand: lane l holds row l % 16, eight places of k from
// 8 * (l / 16) on, and of the results row l % 16 for columns 4 * (l / 16) .. + 3.  A row's scale and zero point are then those of the lane.
// Each wavefront of a work-group has the same rows and a run of k of its own; the sums meet in LDS at the end, in the order of the wavefronts.
//
// Weights, their scales and columns go through a ring of the wavefront's own in LDS that direct loads fill, DEPTH blocks ahead: no barrier before the sums,
// no register for what is under way.  Loads have to come as 64 contiguous bytes to four lanes: with a lane to a row, as MFMAs want them, a CU got 11
// bytes a clock (4096 x 16 x 14336 in 4 bits: 24 us).
//
// 4-bit weights: a block is 128 places, 64 bytes of a row.  Eight codes become numbers by moving nibbles to where a mantissa ends:
//   fp16: the code itself, as a subnormal number (code * 2^-24; MFMAs take those as they are): 7 instructions.
//   bf16: 128 + code, the largest such number with 4 free bits: 9 instructions.
// One MFMA against ones sums the columns' elements of a group; zero point (+ 128) times that comes off the group's sums, which then are multiplied by
// its scale, in fp32.  The sums lose five bits of fp32's 24 to the 128 at most, of which a store to bf16 keeps 8.
// 16-bit weights: a block is 64 places, 128 bytes of a row.
#pragma once

#include <type_traits>

#include "w4.hpp"

namespace mmbo {

namespace stream {

typedef u32x4 __attribute__((aligned(1))) u32x4_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;

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

// Eight numbers from a dword of codes.  Number n stands for (code + kBias) * kUnit.
template <typename T> struct Codes;
template <> struct Codes<half_t> {
    static constexpr float kBias = 0.0f, kUnit = 0x1p-24f;
    struct Masks {};
    __device__ static inline Masks masks() { return Masks{}; }
    __device__ static inline f16x8 expand(uint32_t x, const Masks &)
    {
        union { uint32_t d[4]; f16x8 v; } u;
        const uint32_t even = x & 0x0F0F0F0Fu, odd = x >> 4 & 0x0F0F0F0Fu;
#pragma unroll
        for (int p = 0; p < 4; ++p) u.d[p] = __builtin_amdgcn_perm(odd, even, 0x0c040c00u + p * 0x00010001u);       // byte p of either
        return u.v;
    }
};
template <> struct Codes<bf16_t> {
    static constexpr float kBias = 128.0f, kUnit = 1.0f;
    // (in registers: with both constants in the instruction it would be two)
    struct Masks { uint32_t keep, exponent; };
    __device__ static inline Masks masks()
    {
        Masks m{0x000F000Fu, 0x43004300u};
        asm("" : "+s"(m.keep));
        asm("" : "+v"(m.exponent));
        return m;
    }
    __device__ static inline bf16x8 expand(uint32_t x, const Masks &m)
    {
        union { uint32_t d[4]; bf16x8 v; } u;
        const uint32_t odd = x >> 4;
#pragma unroll
        for (int p = 0; p < 4; ++p) u.d[p] = (__builtin_amdgcn_perm(odd, x, 0x0c040c00u + p * 0x00010001u) & m.keep) | m.exponent;
        return u.v;
    }
};

template <typename T>
__device__ inline typename Type<T>::Frag ones()
{
    const uint32_t one = __is_same(T, half_t) ? 0x3C003C00u : 0x3F803F80u;
    return frag_of<T>(u32x4{one, one, one, one});
}

// 16 bytes a lane from `p` to LDS at lds_addr + 16 * lane; 2 bytes or 1, as a dword, to lds_addr + 4 * lane (lanes that take no part leave theirs as it
// is).  As ring::direct_load16, but from an address a lane: rows may lie anywhere.
__device__ inline void direct_load(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}
__device__ inline void direct_load_u16(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ushort %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}
__device__ inline void direct_load_u8(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}

// Rows of 64 bytes in LDS as direct loads put them: lane l loads chunk (l % 4) ^ (row / 4 % 4) of row l / 4 (of R, then 32 places further).  The exclusive or
// spreads what is read together over the banks: one chunk of 16 rows, or a dword of each of their four chunks.
template <int R>
__device__ inline uint32_t chunk_of_lane(int lane) { return (lane & 3) ^ ((lane >> 2) % R >> 2 & 3); }
__device__ inline uint32_t chunk_at(uint32_t row, uint32_t chunk) { return row * 64 + ((chunk ^ (row >> 2 & 3)) << 4); }

// Columns side by side in LDS: 1, 4, 16 or 32.  Columns in PLANES numbers of type T each, which are added.
template <int N2> constexpr int tiles_of() { return N2 > 16 ? N2 / 16 : 1; }

// Where a lane finds a job's rows of weights in FT tiles of 16, and its columns.  In the place of rows and columns that do not exist: others that do.
template <typename T, int N2, int FT, int PLANES>
struct Job {
    const uint8_t *w[FT];                       // row lane / 4 of codes, or of elements
    const T *scales[FT];                        // row lane % 16
    const uint8_t *zeros[FT];
    const T *x[PLANES][tiles_of<N2>()];         // column lane / 4 % N2 of each tile
    bool x_here[tiles_of<N2>()];                // .. exists
};

// The sums of a wavefront over its share of several jobs: of each job blocks block0 .. block0 + per_job - 1 of k, job after job, and of all these blocks
// numbers first .. first + count - 1.  enter(job, Job &) says where its operands lie, flush(job, sums) takes the sums of what the wavefront had of it.  Results of columns that do not
// exist are not defined.  lds: the wavefront's own LDS_BYTES.
// FOLDS (4-bit weights): times in a block that sums are multiplied by their scale: 1 where groups are whole multiples of 128, 2 of 64, else 4.
template <typename T, bool W4, int N2, int FT, int PLANES, int FOLDS, bool ZEROS, int DEPTH>
struct Stream {
    typedef typename Type<T>::Frag Frag;
    typedef typename Codes<T>::Masks Masks;
    typedef stream::Job<T, N2, FT, PLANES> Job;
    static constexpr int NT = tiles_of<N2>(), BLOCK = W4 ? 128 : 64, STEPS = BLOCK / 32, ROW_BYTES = W4 ? 64 : 128;
    static constexpr int W_LOADS = ROW_BYTES / 64, W_BYTES = FT * W_LOADS * 1024;
    static constexpr int X_LANES = N2 < 16 ? STEPS * N2 * 4 : 64, X_LOADS = N2 < 16 ? 1 : STEPS * NT, X_PLANE = N2 < 16 ? STEPS * N2 * 64 : X_LOADS * 1024;
    static constexpr int X_AT = W_BYTES, S_AT = X_AT + PLANES * X_PLANE, Z_AT = S_AT + (W4 ? FT * 256 : 0), SLOT = Z_AT + (W4 && ZEROS ? FT * 256 : 0);
    static constexpr int LOADS = FT * W_LOADS + PLANES * X_LOADS + (W4 ? FT * (ZEROS ? 2 : 1) : 0);
    static constexpr int LDS_BYTES = (DEPTH * SLOT + 1023) / 1024 * 1024;
    static_assert((DEPTH - 1) * LOADS < 64, "vmcnt counts to 63");
    static_assert(N2 == 1 || N2 == 4 || N2 == 16 || N2 == 32, "");
    typedef f32x4 Sums[NT][FT];

    uint32_t k, group32;                        // places; places of a group / 32
    char *lds;
    int lane;
    uint32_t lds_at, block0, per_job;
    // requests
    Job from;
    uint32_t r_job, r_block, group, rest;       // (group and rest: of the lane's fold)
    // products
    Masks masks;
    struct Operands {
        Frag x[PLANES][STEPS][NT];
        u32x4 w[W4 ? 1 : STEPS][FT];
        uint32_t codes[W4 ? STEPS : 1][FT];
        uint32_t scales[FOLDS][FT], zeros[FOLDS][FT];
    } o;

    __device__ inline Stream(uint32_t k, uint32_t group32, uint32_t block0, uint32_t per_job, char *lds, int lane)
        : k(k), group32(group32), lds(lds), lane(lane), lds_at(__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MMBO_LDS_PTR(lds))), block0(block0),
          per_job(per_job), masks(Codes<T>::masks())
    {
    }
    __host__ __device__ static inline uint32_t blocks_of(uint32_t k) { return (k + BLOCK - 1) / BLOCK; }

    template <typename Enter>
    __device__ inline void enter_job(const Enter &enter)
    {
        enter(r_job, from);
        const uint32_t b = block0 + r_block;
#pragma unroll
        for (int f = 0; f < FT; ++f) from.w[f] += (uint64_t)b * ROW_BYTES + chunk_of_lane<16>(lane) * 16;
        const uint32_t place = b * BLOCK + (N2 < 16 ? lane / (4 * N2) * 32 : 0) + chunk_of_lane<(N2 < 16 ? N2 : 16)>(lane) * 8;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            from.x_here[c] = from.x_here[c] && lane < X_LANES;
#pragma unroll
            for (int q = 0; q < PLANES; ++q) from.x[q][c] += place;
        }
        if constexpr (W4) {
            const uint32_t at = b * 4 + (lane >> 4) * (4 / FOLDS);
            group = at / group32;
            rest = at % group32;
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
        if constexpr (W4) {
            // lane: row lane % 16, fold lane / 16
            const uint32_t g = min(group, (k - 1) / 32 / group32);
            if (lane < 16 * FOLDS)
#pragma unroll
                for (int f = 0; f < FT; ++f) {
                    direct_load_u16(from.scales[f] + g, to + S_AT + f * 256);
                    if constexpr (ZEROS) direct_load_u8(from.zeros[f] + g, to + Z_AT + f * 256);
                }
            group += 4 / group32;
            rest += 4 % group32;
            if (rest >= group32) { rest -= group32; ++group; }
        }
        if ((block0 + r_block) * BLOCK + BLOCK <= k) {
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int h = 0; h < W_LOADS; ++h) direct_load(from.w[f] + h * 64, to + (f * W_LOADS + h) * 1024);
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
#pragma unroll
                for (int j = 0; j < X_LOADS; ++j)
                    if (from.x_here[j % NT]) direct_load(from.x[q][j % NT] + j / NT * 32, to + X_AT + q * X_PLANE + j * 1024);
        } else {
            // The last block of a k that is not a whole number of them: chunks that are there as ever, the others through registers.  Counts of
            // what is under way no longer hold then, so nothing is, for once.
            const int64_t left = (int64_t)k - (block0 + r_block) * BLOCK;
            char *const slot_at = lds + slot * SLOT;
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int h = 0; h < W_LOADS; ++h) {
                    const int64_t here = left - h * 32 - chunk_of_lane<16>(lane) * (W4 ? 32 : 8);
                    u32x4 *const at = reinterpret_cast<u32x4 *>(slot_at + (f * W_LOADS + h) * 1024 + lane * 16);
                    if constexpr (W4) *at = here >= 32 ? *reinterpret_cast<const u32x4_any *>(from.w[f]) : load32_codes(from.w[f], here);
                    else *at = load8(reinterpret_cast<const T *>(from.w[f] + h * 64), here);
                }
#pragma unroll
            for (int q = 0; q < PLANES; ++q)
#pragma unroll
                for (int j = 0; j < X_LOADS; ++j)
                    if (from.x_here[j % NT]) {
                        const int64_t here = left - (N2 < 16 ? lane / (4 * N2) : j / NT) * 32 - chunk_of_lane<(N2 < 16 ? N2 : 16)>(lane) * 8;
                        *reinterpret_cast<u32x4 *>(slot_at + X_AT + q * X_PLANE + j * 1024 + lane * 16) = load8(from.x[q][j % NT] + j / NT * 32, here);
                    }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        ++r_block;
#pragma unroll
        for (int f = 0; f < FT; ++f) from.w[f] += ROW_BYTES;
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
#pragma unroll
            for (int c = 0; c < NT; ++c) from.x[q][c] += BLOCK;
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
                    o.x[q][i][c] = frag_of<T>(*reinterpret_cast<const u32x4 *>(at + X_AT + q * X_PLANE + i * N2 * 64 + chunk_at((lane & (N2 < 16 ? N2 - 1 : 15)) + c * 16, quarter)));
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            if constexpr (W4) {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) o.codes[i][f] = *reinterpret_cast<const uint32_t *>(at + f * 1024 + chunk_at(row, i) + quarter * 4);
#pragma unroll
                for (int q = 0; q < FOLDS; ++q) {
                    o.scales[q][f] = *reinterpret_cast<const uint32_t *>(at + S_AT + f * 256 + (q * 16 + row) * 4);
                    if constexpr (ZEROS) o.zeros[q][f] = *reinterpret_cast<const uint32_t *>(at + Z_AT + f * 256 + (q * 16 + row) * 4);
                }
            } else {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) o.w[i][f] = *reinterpret_cast<const u32x4 *>(at + (f * STEPS + i) * 1024 + chunk_at(row, quarter));
            }
        }
    }

    __device__ inline void multiply(Sums &acc)
    {
        if constexpr (W4) {
#pragma unroll
            for (int q = 0; q < FOLDS; ++q) {
                Sums part;
                f32x4 sums[NT];                  // of the columns' elements
                clear(part);
#pragma unroll
                for (int c = 0; c < NT; ++c) sums[c] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = q * (4 / FOLDS); i < (q + 1) * (4 / FOLDS); ++i) {
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int e = 0; e < PLANES; ++e) sums[c] = Type<T>::mfma(o.x[e][i][c], ones<T>(), sums[c]);
#pragma unroll
                    for (int f = 0; f < FT; ++f) {
                        const Frag w = Codes<T>::expand(o.codes[i][f], masks);
#pragma unroll
                        for (int c = 0; c < NT; ++c)
#pragma unroll
                            for (int e = 0; e < PLANES; ++e) part[c][f] = Type<T>::mfma(o.x[e][i][c], w, part[c][f]);
                    }
                }
#pragma unroll
                for (int f = 0; f < FT; ++f) {
                    // the scale of a number, and the number that stands for 0
                    const float s = (float)__builtin_bit_cast(T, (uint16_t)o.scales[q][f]) * (1.0f / Codes<T>::kUnit);
                    const float z = ((ZEROS ? (float)(o.zeros[q][f] & kW4ZeroMask) : kW4Zero) + Codes<T>::kBias) * Codes<T>::kUnit;
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[c][f][r] = __builtin_fmaf(s, __builtin_fmaf(-z, sums[c][r], part[c][f][r]), acc[c][f][r]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int f = 0; f < FT; ++f)
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int e = 0; e < PLANES; ++e) acc[c][f] = Type<T>::mfma(o.x[e][i][c], frag_of<T>(o.w[i][f]), acc[c][f]);
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

// Tiles of 16 x 16 sums of several wavefronts -> their sum: wavefront after wavefront, in that order.  lds: waves * TILES * 256 floats.  Gives element `at` of
// TILES * 256: column at / 16 % 16, row at % 16 of tile at / 256.
template <int TILES>
__device__ inline void put_sums(float *lds, const f32x4 (&acc)[TILES], int wave, int lane)
{
#pragma unroll
    for (int t = 0; t < TILES; ++t) *reinterpret_cast<f32x4 *>(lds + (wave * TILES + t) * 256 + lane * 4) = acc[t];
}
template <int TILES>
__device__ inline float sum_of(const float *lds, uint32_t at, int waves)
{
    const uint32_t row = at & 15, col = at >> 4 & 15, tile = at >> 8;
    const uint32_t place = tile * 256 + ((col >> 2) * 16 + row) * 4 + (col & 3);
    float v = lds[place];
    for (int w = 1; w < waves; ++w) v += lds[w * TILES * 256 + place];
    return v;
}

}  // namespace stream

// A work-group: 16 * FT rows of W, up to N2 columns of B; its wavefronts share k, a run of blocks each.
template <typename T, int N2, int FT, int FOLDS, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(512)
gemm_w4_stream_kernel(const GemmW4Args a)
{
    using namespace stream;
    typedef Stream<T, true, N2, FT, 1, FOLDS, ZEROS, DEPTH> S;
    constexpr int NT = S::NT, TILES = NT * FT;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint64_t row0 = (uint64_t)blockIdx.x * 16 * FT;
    auto enter = [&](uint32_t, typename S::Job &j) {
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            const uint64_t i = min(row0 + f * 16 + (lane & 15), (uint64_t)a.m - 1);         // (rows past the edge repeat the last one)
            j.w[f] = a.w.q + min(row0 + f * 16 + (lane >> 2), (uint64_t)a.m - 1) * a.w.ldq;
            j.scales[f] = static_cast<const T *>(a.w.scales) + i * a.w.lds;
            j.zeros[f] = a.w.zeros + i * a.w.ldz;
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const uint32_t col = (uint32_t)(lane >> 2) % N2 % 16 + c * 16;
            j.x[0][c] = static_cast<const T *>(a.B) + min(col, a.n - 1) * a.ldb;
            j.x_here[c] = col < a.n;
        }
    };
    f32x4 total[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) total[t] = f32x4{0, 0, 0, 0};
    auto flush = [&](uint32_t, const typename S::Sums &acc) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) total[t] = acc[t / FT][t % FT];
    };
    const uint32_t blocks = S::blocks_of(a.k), each = blocks / waves, more = blocks % waves, count = each + (wave < more);
    S s(a.k, a.group / kW4Group, wave * each + min(wave, more), count, lds + wave * S::LDS_BYTES, lane);
    s.run(0, count, enter, flush);
    __syncthreads();                                                                    // (the sums lie where the rings were)
    float *sums = reinterpret_cast<float *>(lds);
    put_sums<TILES>(sums, total, wave, lane);
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < TILES * 256; at += blockDim.x) {
        const uint32_t tile = at >> 8;
        const uint64_t i = row0 + tile % FT * 16 + (at & 15), j = tile / FT * 16 + (at >> 4 & 15);
        if (i >= a.m || j >= a.n) continue;
        T *c = static_cast<T *>(a.C) + i + j * a.ldc;
        float v = a.alpha * sum_of<TILES>(sums, at, waves);
        if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*c, v);
        *c = (T)v;
    }
}

}  // namespace mmbo
