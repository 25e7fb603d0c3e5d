// A few columns against weights that are read once: a wavefront streams rows of weights past up to 16 columns.
//
// D(column, row) += X(column, l) * W(l, row) on 16x16x32 MFMAs, weights as the second operand: lane l holds row l % 16, eight places of k from
// 8 * (l / 16) on, and of the results row l % 16 for columns 4 * (l / 16) .. + 3.  A row's scale and zero point are then those of the lane.
// Each wavefront of a work-group has the same rows and a run of k of its own; the sums meet in LDS at the end, in the order of the wavefronts.
//
// Weights and columns go through a ring of the wavefront's own in LDS that direct loads fill, DEPTH blocks ahead: no barrier before the sums, no register
// for what is under way.  Loads have to come as 64 contiguous bytes to four lanes: with a lane to a row, as MFMAs want them, a CU got 11 bytes a
// clock of the columns it needs beside the weights (16 x 4096 x 14336: 24 us).
//
// 4-bit weights: a block is 128 places, 64 bytes of a row.  Eight codes become numbers by moving nibbles to where a mantissa ends:
//   fp16: the code itself, as a subnormal number (code * 2^-24; MFMAs take those as they are): 7 instructions.
//   bf16: 128 + code, the largest such number with 4 free bits: 9 instructions.
// One MFMA against ones sums the columns' elements of a group; zero point (+ 128) times that comes off the group's sums, which then are multiplied by
// its scale, in fp32.  The sums lose five bits of fp32's 24 to the 128 at most, of which a store to bf16 keeps 8.
#pragma once

#include <type_traits>

#include "w4.hpp"

namespace mmbo {

namespace stream {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
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
// Eight codes from `p`, of which `here` exist; the others may be anything.
__device__ inline uint32_t load8_codes(const uint8_t *p, int64_t here)
{
    if (here >= 8) return *reinterpret_cast<const u32_any *>(p);
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (2 * i < here) v |= (uint32_t)p[i] << (8 * i);
    return v;
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

// 16 bytes a lane from `p` to LDS at lds_addr + 16 * lane (lanes that take no part leave theirs as it is).  As ring::direct_load16, but from an address a
// lane: rows may lie anywhere.
__device__ inline void direct_load(const void *p, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds_addr) : "memory");
}

// R rows of 64 bytes in LDS as direct loads put them: lane l loads chunk (l % 4) ^ (row / 4 % 4) of row l / 4 % R.  The exclusive or spreads what is read together
// over the banks: one chunk of 16 rows, or a dword of each of their four chunks.
template <int R>
__device__ inline uint32_t chunk_of_lane(int lane) { return (lane & 3) ^ ((lane >> 2) % R >> 2 & 3); }
__device__ inline uint32_t chunk_at(uint32_t row, uint32_t chunk) { return row * 64 + ((chunk ^ (row >> 2 & 3)) << 4); }

// A lane's rows of weights in FT tiles of 16 rows, and its columns.  Rows and columns that do not exist: others that do.
template <typename T, int FT>
struct Lane {
    const uint8_t *w[FT], *w_end[FT];           // rows lane / 4 and lane % 16 of codes, or of elements
    const T *scales[FT];                        // row lane % 16
    const uint8_t *zeros[FT];
    const T *x, *x_end;                         // columns lane / 4 % N2 and lane % 16
    bool x_here;                                // column lane / 4 % N2 exists
    uint32_t k, group32;                        // places; places of a group / 32
};

// The sums of a wavefront over its share of k, 4-bit weights: `count` blocks of 128 places from block `first` on; with `tail` also what k leaves behind its
// whole blocks.  Results of columns that do not exist are not defined.  lds: the wavefront's own LDS_BYTES.
// FOLDS: times in a block that sums are multiplied by their scale: 1 where groups are whole multiples of 128, 2 of 64, else 4.
template <typename T, int N2, int FT, int FOLDS, int DEPTH>
struct Stream4 {
    typedef typename Type<T>::Frag Frag;
    typedef typename Codes<T>::Masks Masks;
    static constexpr int BLOCK = 128;
    static constexpr int W_BYTES = FT * 1024, SLOT = W_BYTES + N2 * 256, X_LOADS = N2 < 4 ? 1 : N2 / 4, LOADS = FT + X_LOADS;
    static constexpr int SCALES = 8 * FOLDS;    // groups whose scales lie in LDS at a time
    static constexpr int LDS_BYTES = DEPTH * SLOT + SCALES * FT * 16 * 8;
    static_assert((DEPTH - 1) * LOADS < 64, "vmcnt counts to 63");

    struct Scale { float s, z; };               // the scale of a number, and the number that stands for 0
    __device__ static inline Scale scale_of(T scale, float zero)
    {
        return Scale{(float)scale * (1.0f / Codes<T>::kUnit), (zero + Codes<T>::kBias) * Codes<T>::kUnit};
    }
    __device__ static inline Scale scale_of(const Lane<T, FT> &p, int f, uint32_t g)
    {
        return scale_of(p.scales[f][g], p.zeros[f] ? (float)(p.zeros[f][g] & kW4ZeroMask) : kW4Zero);
    }
    // part: the sums of a group's places, sums: of its columns' elements
    __device__ static inline void fold(f32x4 (&acc)[FT], const f32x4 (&part)[FT], const f32x4 &sums, const Scale (&s)[FT])
    {
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[f][r] = __builtin_fmaf(s[f].s, __builtin_fmaf(-s[f].z, sums[r], part[f][r]), acc[f][r]);
    }
    __device__ static inline void products(f32x4 (&part)[FT], f32x4 &sums, const Frag &x, const uint32_t (&codes)[FT], const Masks &masks)
    {
        sums = Type<T>::mfma(x, ones<T>(), sums);
#pragma unroll
        for (int f = 0; f < FT; ++f) part[f] = Type<T>::mfma(x, Codes<T>::expand(codes[f], masks), part[f]);
    }
    __device__ static inline void clear(f32x4 (&part)[FT], f32x4 &sums)
    {
        sums = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < FT; ++f) part[f] = f32x4{0, 0, 0, 0};
    }

    __device__ static inline void run(f32x4 (&acc)[FT], const Lane<T, FT> &p, uint32_t first, uint32_t count, bool tail, char *lds, int lane)
    {
        const uint32_t row = lane & 15, quarter = lane >> 4;
        const Masks masks = Codes<T>::masks();
        const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MMBO_LDS_PTR(lds));
        const uint8_t *w[FT];
#pragma unroll
        for (int f = 0; f < FT; ++f) w[f] = p.w[f] + (uint64_t)first * 64 + chunk_of_lane<16>(lane) * 16;
        const T *x = p.x + (uint64_t)first * BLOCK + lane / (4 * N2) * 32 + chunk_of_lane<N2>(lane) * 8;
        auto request = [&](uint32_t slot) {
            const uint32_t to = lds_at + slot * SLOT;
#pragma unroll
            for (int f = 0; f < FT; ++f) {
                direct_load(w[f], to + f * 1024);
                w[f] += 64;
            }
            if (p.x_here)
#pragma unroll
                for (int j = 0; j < X_LOADS; ++j) direct_load(x + j * (16 / N2) * 32, to + W_BYTES + j * 1024);
            x += BLOCK;
        };
#pragma unroll
        for (int s = 0; s < DEPTH; ++s)
            if ((uint32_t)s < count) request(s);

        if (tail && p.k % BLOCK != 0) {                                          // what is left of k, while the ring fills
            uint32_t codes[4][FT];
            Frag xs[4];
            Scale sc[4][FT];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t l0 = p.k / BLOCK * BLOCK + i * 32, l = l0 + quarter * 8;
                const int64_t here = (int64_t)p.k - l;
#pragma unroll
                for (int f = 0; f < FT; ++f) {
                    codes[i][f] = load8_codes(p.w_end[f] + l / 2, here);
                    sc[i][f] = scale_of(p, f, min(l0, p.k - 1) / 32 / p.group32);
                }
                xs[i] = frag_of<T>(load8(p.x_end + l, here));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 part[FT], sums;
                clear(part, sums);
                products(part, sums, xs[i], codes[i], masks);
                fold(acc, part, sums, sc[i]);
            }
        }

        Scale *const scales = reinterpret_cast<Scale *>(lds + DEPTH * SLOT);     // [group - group0][row]
        uint32_t group0 = first * 4 / p.group32, rest = first * 4 % p.group32, group = 0;
        const uint32_t last = count ? ((first + count) * 4 - 1) / p.group32 : 0;
        auto load_scales = [&] {
            for (uint32_t g = quarter; g < SCALES && group0 + g <= last; g += 4)
#pragma unroll
                for (int f = 0; f < FT; ++f) scales[(g * FT + f) * 16 + row] = scale_of(p, f, group0 + g);
        };
        if (count) load_scales();

        struct Operands {
            Frag x[4];
            uint32_t codes[4][FT];
        } o;
        auto read = [&](uint32_t slot) {
            const char *const at = lds + slot * SLOT;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o.x[i] = frag_of<T>(*reinterpret_cast<const u32x4 *>(at + W_BYTES + i * N2 * 64 + chunk_at(lane & (N2 - 1), quarter)));
#pragma unroll
                for (int f = 0; f < FT; ++f) o.codes[i][f] = *reinterpret_cast<const uint32_t *>(at + f * 1024 + chunk_at(row, i) + quarter * 4);
            }
        };
        auto multiply = [&] {
#pragma unroll
            for (int q = 0; q < FOLDS; ++q) {
                f32x4 part[FT], sums;
                Scale s[FT];
#pragma unroll
                for (int f = 0; f < FT; ++f) s[f] = scales[(group * FT + f) * 16 + row];
                clear(part, sums);
#pragma unroll
                for (int i = q * (4 / FOLDS); i < (q + 1) * (4 / FOLDS); ++i) products(part, sums, o.x[i], o.codes[i], masks);
                fold(acc, part, sums, s);
                rest += 4 / FOLDS;
                if (rest >= p.group32) {                                         // (a group is no shorter than what is folded at once)
                    rest -= p.group32;
                    if (++group == SCALES) {
                        group0 += SCALES;
                        group = 0;
                        load_scales();
                    }
                }
            }
        };
        // (the compiler does not count direct loads; the "memory" clobbers keep what is read between them)
        uint32_t slot = 0, s = 0;
        for (; s + DEPTH < count; ++s) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * LOADS) : "memory");
            read(slot);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                   // in registers: the slot is free
            request(slot);
            multiply();
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (; s < count; ++s) {
            read(slot);
            multiply();
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
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
template <typename T, int N2, int FT, int FOLDS, int DEPTH>
__global__ void __launch_bounds__(FT > 1 ? 512 : 1024)
gemm_w4_stream_kernel(const GemmW4Args a)
{
    using namespace stream;
    typedef Stream4<T, N2, FT, FOLDS, DEPTH> S;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint64_t row0 = (uint64_t)blockIdx.x * 16 * FT;
    Lane<T, FT> p;
#pragma unroll
    for (int f = 0; f < FT; ++f) {
        const uint64_t i = min(row0 + f * 16 + (lane & 15), (uint64_t)a.m - 1);         // (rows past the edge repeat the last one)
        p.w[f] = a.w.q + min(row0 + f * 16 + (lane >> 2), (uint64_t)a.m - 1) * a.w.ldq;
        p.w_end[f] = a.w.q + i * a.w.ldq;
        p.scales[f] = static_cast<const T *>(a.w.scales) + i * a.w.lds;
        p.zeros[f] = a.w.zeros ? a.w.zeros + i * a.w.ldz : nullptr;
    }
    const T *B = static_cast<const T *>(a.B);
    p.x = B + min((uint32_t)(lane >> 2) % N2, a.n - 1) * a.ldb;
    p.x_here = (uint32_t)(lane >> 2) % N2 < a.n && lane < N2 * 16;
    p.x_end = B + min((uint32_t)lane & 15, a.n - 1) * a.ldb;
    p.k = a.k;
    p.group32 = a.group / kW4Group;
    f32x4 acc[FT];
#pragma unroll
    for (int f = 0; f < FT; ++f) acc[f] = f32x4{0, 0, 0, 0};
    const uint32_t blocks = a.k / S::BLOCK, each = blocks / waves, more = blocks % waves;
    S::run(acc, p, wave * each + min(wave, more), each + (wave < more), wave == waves - 1, lds + wave * S::LDS_BYTES, lane);
    __syncthreads();                                                                    // (the sums lie where the rings were)
    float *sums = reinterpret_cast<float *>(lds);
    put_sums<FT>(sums, acc, wave, lane);
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < FT * 256; at += blockDim.x) {
        const uint64_t i = row0 + (at >> 8) * 16 + (at & 15), j = at >> 4 & 15;
        if (i >= a.m || j >= a.n) continue;
        T *c = static_cast<T *>(a.C) + i + j * a.ldc;
        float v = a.alpha * sum_of<FT>(sums, at, waves);
        if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*c, v);
        *c = (T)v;
    }
}

}  // namespace mmbo
