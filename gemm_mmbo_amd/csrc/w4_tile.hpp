// Products with 4-bit weights and many columns: tiles of 32 * WM rows by 16 * NC columns, a wavefront to 32 rows.
//
// A wavefront expands its own rows' codes -- no row's is expanded twice in a work-group -- and multiplies them with all of the tile's columns, on the
// MFMAs and in the layout of stream.hpp.  Codes, scales and columns go through a ring of DEPTH slots of 128 places in LDS that direct loads fill, one barrier
// a slot.  A code becomes the exact number code - zero:
//   fp16: times 2^-10, as in stream.hpp: 11 instructions for eight.
//   bf16: from the subnormal fp16 number code * 2^-24 one mixed-precision fma makes code - zero in fp32, and two of those are packed: 19.
// A group's sums, in fp32, are multiplied by its scale and added to the total.  What bounds it is the issue of vector instructions beside the MFMAs: 16
// MFMAs of 16 clocks a step of 32 places, and for those two wavefronts of a SIMD 2 * (38 (fp16: 22) + 16 + 16) issues of 4.
// 8192 x 2048 x 4096 in groups of 128: fp16 136 us, bf16 147, 1.0 and 0.94 PFLOP/s; groups of 64 151 and 163, of 32 169 (fp16).
#pragma once

#include "stream.hpp"

namespace mmbo {

namespace tile {

using namespace stream;

constexpr int BLOCK = 128, STEPS = 4;

template <typename T, int WM, int NC, int FOLDS, bool ZEROS, int DEPTH>
struct Config {
    static constexpr int ROWS = 32 * WM, COLUMNS = 16 * NC, THREADS = 64 * WM;
    static constexpr int X_LOADS = 4 * NC / WM,           // of whole lines: eight columns of 64 places each
                          LOADS = X_LOADS + 2 + (ZEROS ? 4 : 2);
    static constexpr int W_AT = 2 * COLUMNS * 128, S_TILE = 64 * FOLDS, S_AT = W_AT + ROWS * 64, Z_AT = S_AT + WM * 2 * S_TILE,
                         SLOT = (Z_AT + (ZEROS ? WM * 2 * S_TILE : 0) + 1023) / 1024 * 1024;
    static constexpr int LDS_BYTES = DEPTH * SLOT;
    static constexpr bool FITS = LDS_BYTES <= (int)kLds;
    static_assert(4 * NC % WM == 0 && DEPTH == 3, "");
};

}  // namespace tile

template <typename T, int WM, int NC, int FOLDS, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(64 * WM, WM > 4 ? 2 : 1)
gemm_w4_tile_kernel(const GemmW4Args a)
{
    using namespace tile;
    typedef Config<T, WM, NC, FOLDS, ZEROS, DEPTH> C;
    typedef typename Type<T>::Frag Frag;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, quarter = lane >> 4;
    const uint32_t lds_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MMBO_LDS_PTR(lds));
    // (tiles of one run of rows one after the other on an XCD: their weights are then in its cache)
    uint32_t wg0, wg1;
    {
        const uint32_t rows = (uint32_t)((a.m + C::ROWS - 1) / C::ROWS), columns = (a.n + C::COLUMNS - 1) / C::COLUMNS;
        wg_remap(blockIdx.x, rows, columns, 8, 8, wg0, wg1);
    }
    const uint64_t row0 = (uint64_t)wg0 * C::ROWS + wave * 32, col0 = (uint64_t)wg1 * C::COLUMNS;
    const uint64_t last_row = a.m - 1, last_col = a.n - 1;         // (what lies past the edge repeats the last ones)

    const uint8_t *w[2], *zeros[2];
    const T *scales[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        w[f] = a.w.q + min(row0 + f * 16 + (lane >> 2), last_row) * a.w.ldq + chunk_of<64>(lane >> 2, lane) * 16;
        const uint64_t i = min(row0 + f * 16 + row, last_row);
        scales[f] = static_cast<const T *>(a.w.scales) + i * a.w.lds;
        zeros[f] = ZEROS ? a.w.zeros + i * a.w.ldz : nullptr;
    }
    // load j of this wavefront: eight columns (first + j) % (2 * NC) of line (first + j) / (2 * NC)
    constexpr int EIGHTS = 2 * NC, X_COLS = C::X_LOADS < EIGHTS ? C::X_LOADS : EIGHTS;
    const uint32_t x_first = wave * C::X_LOADS;
    auto x_column = [&](int j) { return (x_first + j) % EIGHTS * 8 + (lane >> 3); };
    auto x_chunk = [&](int j) { return chunk_of<128>(x_column(j), lane); };
    const T *x[X_COLS];
#pragma unroll
    for (int j = 0; j < X_COLS; ++j)
        x[j] = static_cast<const T *>(a.B) + min(col0 + x_column(j), last_col) * a.ldb + x_first / EIGHTS * 64 + x_chunk(j) * 8;

    const uint32_t slots = (a.k + BLOCK - 1) / BLOCK, group32 = a.group / kW4Group, last_group = (a.k - 1) / a.group;
    uint32_t group, rest;
    {
        const uint32_t at = quarter * (4 / FOLDS);
        group = at / group32;
        rest = at % group32;
    }
    auto request = [&](uint32_t s, uint32_t buffer) {
        const uint32_t to = lds_at + buffer * C::SLOT;
        const uint32_t g = min(group, last_group);
        if (lane < 16 * FOLDS)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                direct_load_u16(scales[f] + g, to + C::S_AT + (wave * 2 + f) * C::S_TILE);
                if constexpr (ZEROS) direct_load_u8(zeros[f] + g, to + C::Z_AT + (wave * 2 + f) * C::S_TILE);
            }
        group += 4 / group32;
        rest += 4 % group32;
        if (rest >= group32) { rest -= group32; ++group; }
        if (s * BLOCK + BLOCK <= a.k) {
#pragma unroll
            for (int f = 0; f < 2; ++f) direct_load(w[f], to + C::W_AT + (wave * 2 + f) * 1024);
            ring::static_for<C::X_LOADS>([&](auto J) {
                constexpr int j = decltype(J)::value;
                direct_load<j / EIGHTS * 128>(x[j % X_COLS], to + (x_first + j) * 1024);
            });
        } else {
            // The last slot of a k that is not a whole number of them: through registers, and nothing is under way for once.
            const int64_t left = (int64_t)a.k - s * BLOCK;
            char *const at = lds + buffer * C::SLOT;
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int64_t here = left - chunk_of<64>(lane >> 2, lane) * 32;
                *reinterpret_cast<u32x4 *>(at + C::W_AT + (wave * 2 + f) * 1024 + lane * 16) = here >= 32 ? *reinterpret_cast<const u32x4_any *>(w[f]) : load32_codes(w[f], here);
            }
#pragma unroll
            for (int j = 0; j < C::X_LOADS; ++j) {
                const int64_t here = left - (x_first + j) / EIGHTS * 64 - x_chunk(j) * 8;
                *reinterpret_cast<u32x4 *>(at + (x_first + j) * 1024 + lane * 16) = load8(x[j % X_COLS] + j / EIGHTS * 64, here);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) w[f] += 64;
#pragma unroll
        for (int j = 0; j < X_COLS; ++j) x[j] += BLOCK;
    };

    f32x4 acc[2][NC];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[f][c] = f32x4{0, 0, 0, 0};
    auto multiply = [&](uint32_t buffer) {
        const char *const at = lds + buffer * C::SLOT;
#pragma unroll
        for (int q = 0; q < FOLDS; ++q) {
            float scale[2];
            typename Codes<T, true>::Zero zero[2];
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                scale[f] = (float)__builtin_bit_cast(T, *reinterpret_cast<const uint16_t *>(at + C::S_AT + (wave * 2 + f) * C::S_TILE + (q * 16 + row) * 4)) * (1.0f / Codes<T, true>::kUnit);
                zero[f] = Codes<T, true>::zero_of(ZEROS ? *reinterpret_cast<const uint32_t *>(at + C::Z_AT + (wave * 2 + f) * C::S_TILE + (q * 16 + row) * 4) & kW4ZeroMask : (uint32_t)kW4Zero);
            }
            f32x4 part[2][NC];
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int c = 0; c < NC; ++c) part[f][c] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = q * (4 / FOLDS); i < (q + 1) * (4 / FOLDS); ++i) {
                Frag wf[2];
#pragma unroll
                for (int f = 0; f < 2; ++f)
                    wf[f] = Codes<T, true>::expand(*reinterpret_cast<const uint32_t *>(at + C::W_AT + (wave * 2 + f) * 1024 + chunk_at<64>(row, i) + quarter * 4), zero[f]);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const Frag xf = frag_of<T>(*reinterpret_cast<const u32x4 *>(at + (i / 2 * NC + c) * 2048 + chunk_at<128>(row, i % 2 * 4 + quarter)));
#pragma unroll
                    for (int f = 0; f < 2; ++f) part[f][c] = Type<T>::mfma(xf, wf[f], part[f][c]);
                }
            }
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[f][c][r] = __builtin_fmaf(scale[f], part[f][c][r], acc[f][c][r]);
            // (Two groups' sums side by side take more registers than there are: 8192 x 2048 x 4096 in fp16 and groups of 64 took 214 us, with them apart 151.  The
            // compiler keeps four of them apart by itself, and then orders them better: 166 us against 173.)
            if constexpr (FOLDS == 2) __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Slot s is complete when every wavefront has waited for its own part of it: the barrier.  Behind it all are also done with slot s - 1, whose buffer
    // takes slot s + 2.
    if (slots > 0) request(0, 0);
    if (slots > 1) request(1, 1);
    uint32_t buffer = 0;
    for (uint32_t s = 0; s < slots; ++s) {
        if (s + 1 < slots) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(C::LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 2 < slots) request(s + 2, buffer == 0 ? 2 : buffer - 1);
        multiply(buffer);
        buffer = buffer == 2 ? 0 : buffer + 1;
    }

#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint64_t i = row0 + f * 16 + row, j = col0 + c * 16 + quarter * 4 + r;
                if (i >= a.m || j >= a.n) continue;
                T *to = static_cast<T *>(a.C) + i + j * a.ldc;
                float v = a.alpha * acc[f][c][r];
                if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*to, v);
                *to = (T)v;
            }
}

}  // namespace mmbo
