// C ABI of the products with 4-bit weights and of their format: argument checks and dispatch; quantize and dequantize.
#include "../../include/mmbo_gemm.h"

#include <algorithm>
#include <type_traits>

#include "w4_tile.hpp"

namespace mmbo {
namespace {

template <typename T>
__device__ inline float load_scale(const void *p, uint64_t at) { return (float)static_cast<const T *>(p)[at]; }

template <typename T> struct Limits;
template <> struct Limits<float> { static constexpr float largest = 3.40282346638528859812e38f; };
template <> struct Limits<half_t> { static constexpr float largest = 65504.0f; };
template <> struct Limits<bf16_t> { static constexpr float largest = 3.38953138925153547590e38f; };

// w as the format counts it: NaN is 0, an infinity the largest finite number
template <typename TW>
__device__ inline float finite(float w)
{
    const float most = Limits<TW>::largest;
    return w != w ? 0.0f : __builtin_amdgcn_fmed3f(w, -most, most);
}

// The whole number nearest to w / s, halves to even, for numbers within 16 or clamped there; by = 1 / s.  The product's rounding may pick the wrong one next to a
// border; the remainder w - n * s, which is exact in fp32, says so.
__device__ inline float nearest(float w, float s, float by)
{
    float n = rintf(__builtin_amdgcn_fmed3f(w * by, -16.0f, 16.0f));
    const float r = __builtin_fmaf(-n, s, w), half = 0.5f * s;
    if (__builtin_fabsf(r) >= half) {                               // (rare)
        const bool odd = ((int)n & 1) != 0;
        if (r > half || (r == half && odd)) n += 1.0f;
        else if (r < -half || (r == -half && odd)) n -= 1.0f;
    }
    return n;
}

// Sixteen bytes or the elements of them that exist (any number); the others are 0.
template <typename TW> constexpr int kPer16 = 16 / (int)sizeof(TW);
using stream::u32x4_any;
using stream::u32_any;
template <typename TW>
__device__ inline u32x4 load_part(const TW *p, int64_t here)
{
    if (here >= kPer16<TW>) return *reinterpret_cast<const u32x4_any *>(p);
    union { u32x4 q; TW e[kPer16<TW>]; } u;
    u.q = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kPer16<TW> - 1; ++i)
        if (i < here) u.e[i] = p[i];
    return u.q;
}

// LANES lanes, neighbours, have a group of a row: 16 elements each, 16 bytes at a time.  Groups of up to 64 * 16 elements go by in one step and are read once; longer
// ones are read twice, the second time from the cache.
// Bound by what it reads and writes, as long as the instructions for an element are few: a division of 64 bits for each 16 bytes' place, a branch for each element's
// rounding made it 69 us for 8192 x 8192 in bf16, groups of 128, whose 168 MB take 33; this is 45 us.
constexpr int kQuantElements = 16;
template <typename TW, typename T, int LANES>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const QuantArgs a)
{
    constexpr int E = kPer16<TW>, PIECES = kQuantElements / E;
    const uint32_t at = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const uint32_t i = at / a.groups, g = at - i * a.groups;
    if (i >= a.m) return;                                           // (the lanes of a group together)
    const uint32_t l0 = g * a.group, length = min(a.group, a.k - l0);
    const TW *w = static_cast<const TW *>(a.W) + i * a.ldw + l0;
    float low = 0.0f, high = 0.0f, v[PIECES][E];
    auto load = [&](uint32_t step) {
        union { u32x4 q; TW e[E]; } u[PIECES];
        if (step + LANES * kQuantElements <= length) {              // (all pieces under way together)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) u[p].q = *reinterpret_cast<const u32x4_any *>(w + step + (p * LANES + lane) * E);
        } else {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) u[p].q = load_part<TW>(w + step + (p * LANES + lane) * E, (int64_t)length - (step + (p * LANES + lane) * E));
        }
        // (what is finite times 0 is 0, and their sum says so at an instruction an element; one that is not is rare)
        float nothing = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[p][e] = (float)u[p].e[e];
                nothing = __builtin_fmaf(v[p][e], 0.0f, nothing);
            }
        if (nothing != nothing)
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int e = 0; e < E; ++e) v[p][e] = finite<TW>(v[p][e]);
    };
    for (uint32_t step = 0; step < length; step += LANES * kQuantElements) {
        load(step);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                low = fminf(low, v[p][e]);
                high = fmaxf(high, v[p][e]);
            }
    }
    for (int d = 1; d < LANES; d <<= 1) {
        low = fminf(low, __shfl_xor(low, d));
        high = fmaxf(high, __shfl_xor(high, d));
    }
    const bool zeros = a.w.zeros != nullptr;
    // (in 64 bits: high - low may pass the largest float)
    float s = zeros ? (float)(((double)high - (double)low) / 15.0) : fmaxf(high, -low) / 7.0f;
    s = (float)(T)fminf(s, Limits<T>::largest);
    float z = zeros ? 0.0f : kW4Zero;
    // (scales so small that 1 / s is infinite: as everything by 2^64, which changes no quotient; without a scale every number is the zero point)
    const float up = s < 0x1p-100f ? 0x1p64f : 1.0f, su = s * up, by = s == 0.0f ? 0.0f : 1.0f / su;
    const float half = s == 0.0f ? __builtin_inff() : 0.5f * su;
    if (zeros && s != 0.0f) z = fminf(fmaxf(nearest(-low * up, su, by), 0.0f), 15.0f);
    if (lane == 0) {
        static_cast<T *>(const_cast<void *>(a.w.scales))[g + i * a.w.lds] = (T)s;
        if (zeros) const_cast<uint8_t *>(a.w.zeros)[g + i * a.w.ldz] = (uint8_t)z;
    }
    uint8_t *q = const_cast<uint8_t *>(a.w.q) + i * a.w.ldq + l0 / 2;
    const bool once = length <= LANES * kQuantElements;
    for (uint32_t step = 0; step < length; step += LANES * kQuantElements) {
        if (!once) load(step);
        float n[PIECES][E], worst = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[p][e] *= up;
                n[p][e] = rintf(__builtin_amdgcn_fmed3f(v[p][e] * by, -16.0f, 16.0f));
                worst = fmaxf(worst, __builtin_fabsf(__builtin_fmaf(-n[p][e], su, v[p][e])));
            }
        if (worst >= half)                                          // (one of them on a border, or next to it)
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int e = 0; e < E; ++e) n[p][e] = nearest(v[p][e], su, by);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t l = step + (p * LANES + lane) * E;
            if (l >= length) continue;
            uint32_t codes = 0;
#pragma unroll
            for (int e = 0; e < E; e += 2) {                        // two codes are a byte
                const float c0 = __builtin_amdgcn_fmed3f(n[p][e] + z, 0.0f, 15.0f), c1 = __builtin_amdgcn_fmed3f(n[p][e + 1] + z, 0.0f, 15.0f);
                codes = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(c1, 16.0f, c0), e / 2, codes);
            }
            const uint32_t here = min(length - l, (uint32_t)E);
            typedef uint16_t __attribute__((aligned(1))) u16_any;
            if (here == E) {
                if constexpr (E == 8) *reinterpret_cast<u32_any *>(q + l / 2) = codes;
                else *reinterpret_cast<u16_any *>(q + l / 2) = (uint16_t)codes;
            } else {
                codes &= (1u << (4 * here)) - 1;
                for (uint32_t b = 0; b < (here + 1) / 2; ++b) q[l / 2 + b] = (uint8_t)(codes >> (8 * b));
            }
        }
    }
}

// Four threads have 32 places of a row, with one scale.  Bound by what it reads and writes: 8192 x 8192 in groups of 128, 168 MB, 30 us (5.6 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const QuantArgs a)
{
    const uint32_t pieces = (a.k + 31) / 32;
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (uint64_t)a.m * pieces * 4) return;
    // (four threads to a piece, eight places each: 64 bytes of W leave together)
    const uint64_t piece = at >> 2, i = piece / pieces;
    const uint32_t p = (uint32_t)(piece - i * pieces), g = p * 32 / a.group, l = p * 32 + (uint32_t)(at & 3) * 8;
    if (l >= a.k) return;
    const float z = a.w.zeros ? (float)(a.w.zeros[g + i * a.w.ldz] & kW4ZeroMask) : kW4Zero, s = load_scale<T>(a.w.scales, g + i * a.w.lds);
    const uint8_t *q = a.w.q + i * a.w.ldq + l / 2;
    T *to = static_cast<T *>(a.W) + i * a.ldw + l;
    union { u32x4 v; T e[8]; } u;
    if (l + 8 <= a.k) {
        const uint32_t codes = *reinterpret_cast<const u32_any *>(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) u.e[e] = (T)(((float)(codes >> (4 * e) & 15) - z) * s);
        *reinterpret_cast<u32x4_any *>(to) = u.v;
    } else {
        for (uint32_t e = 0; l + e < a.k; ++e) to[e] = (T)(((float)(e & 1 ? q[e / 2] >> 4 : q[e / 2] & 15) - z) * s);
    }
}

// What the three calls check of a weight's sizes.
int check_weight(size_t m, size_t k, size_t group, size_t ldq, size_t lds, const void *zeros, size_t ldz)
{
    if (m > kMaxDim || k > kMaxDim || ldq > kMaxDim || lds > kMaxDim) return MMBO_ERR_INVALID_SIZE;
    if (group == 0 || group % kW4Group != 0 || group > kMaxDim) return MMBO_ERR_INVALID_SIZE;
    const size_t groups = (k + group - 1) / group;
    if (ldq % 2 != 0 || ldq < k || lds < groups) return MMBO_ERR_INVALID_SIZE;
    if (zeros && (ldz > kMaxDim || ldz < groups)) return MMBO_ERR_INVALID_SIZE;
    return MMBO_OK;
}

W4Matrix matrix_of(const void *Q, size_t ldq, const void *scales, size_t lds, const unsigned char *zeros, size_t ldz)
{
    return W4Matrix{static_cast<const uint8_t *>(Q), scales, zeros, (uint64_t)ldq / 2, (uint64_t)lds, (uint64_t)ldz};
}

int status_of(hipError_t e) { return e == hipSuccess ? MMBO_OK : report_hip_error(e); }

// launch(first row, rows) over all rows, so many at a time that their threads, `threads` a row, are fewer than the 2^32 of a grid.
template <typename Launch>
int by_rows(size_t m, size_t threads, const Launch &launch)
{
    const size_t most = std::max<size_t>((1ull << 31) / threads, 1);
    for (size_t i = 0; i < m; i += most)
        if (hipError_t e = launch(i, std::min(m - i, most))) return report_hip_error(e);
    return MMBO_OK;
}

constexpr int kStreamWaves = 8;

template <typename T, int N2, int FT, int FOLD, bool ZEROS>
hipError_t launch_stream_kernel(const GemmW4Args &a, hipStream_t s)
{
    // Blocks under way in a ring.  Work-groups beside each other on a CU hide what a deeper ring would, and need the LDS: 28672 x 1 x 8192 31.5 us with rings of 2, 3 and
    // 4 (work-groups of sixteen wavefronts took a seventh longer); rings of 2, 3 and 4: 4096 x 16 x 14336 13.5, 14.0 and 14.6 us, 8192 x 64 x 8192 27.1, 28.5 and 36.1.
    constexpr int DEPTH = N2 == 1 ? 3 : 2;
    typedef stream::Stream<T, true, N2, FT, 1, FOLD, ZEROS, DEPTH> S;
    constexpr int kWaveBytes = S::LDS_BYTES + 2 * S::SET_FLOATS * 4, kMost = std::min<int>(kStreamWaves, kLds / kWaveBytes);
    static std::atomic<bool> set[64];
    auto kernel = gemm_w4_stream_kernel<T, N2, FT, FOLD, ZEROS, DEPTH>;
    if (hipError_t e = allow_lds(kernel, set)) return e;
    const int waves = (int)std::max<uint32_t>(std::min<uint32_t>(S::blocks_of(a.k), kMost), 1);
    // as many work-groups as the CUs hold at a time, two of eight wavefronts each at most (128256 x 1 x 4096: one 68, two 58, three 58 us)
    const unsigned columns = (unsigned)ceil_div(a.n, N2), held = 256 * std::min<unsigned>(kLds / (waves * kWaveBytes), 2 * kStreamWaves / waves);
    const unsigned groups = (unsigned)std::min<size_t>(ceil_div(a.m, 16 * FT), std::max(held / columns, 1u));
    return launch_args(kernel, dim3(groups, columns), dim3(waves * 64), waves * kWaveBytes, s, a);
}

template <typename T, int N2, int FT, int FOLD>
hipError_t launch_stream_folds(const GemmW4Args &a, hipStream_t s)
{
    return a.w.zeros ? launch_stream_kernel<T, N2, FT, FOLD, true>(a, s) : launch_stream_kernel<T, N2, FT, FOLD, false>(a, s);
}

template <typename T, int N2, int FT>
hipError_t launch_stream_tile(const GemmW4Args &a, hipStream_t s)
{
    if (a.group % 128 == 0) return launch_stream_folds<T, N2, FT, 128>(a, s);
    if (a.group % 64 == 0) return launch_stream_folds<T, N2, FT, 64>(a, s);
    return launch_stream_folds<T, N2, FT, 32>(a, s);
}

template <typename T, int N2>
hipError_t launch_stream_columns(const GemmW4Args &a, hipStream_t s)
{
    // Two tiles of rows a work-group where that still is a work-group for each of 256 CUs: the columns, which every work-group reads, are then read half as
    // often.  8192 x 16 x 8192 12.2 us beside 12.4, 14336 x 4 x 4096 9.4 beside 9.8, 128256 x 1 x 4096 58 beside 63; 4096 x 16 x 14336 16.7 beside 13.1.
    return a.m >= 256 * 32 ? launch_stream_tile<T, N2, 2>(a, s) : launch_stream_tile<T, N2, 1>(a, s);
}

template <typename T, int WM, int NC, int FOLDS, bool ZEROS>
hipError_t launch_tile_kernel(const GemmW4Args &a, hipStream_t s)
{
    typedef tile::Config<T, WM, NC, FOLDS, ZEROS, 3> C;
    if constexpr (!C::FITS) {                    // (eight wavefronts with four scales and zero points a slot)
        return launch_tile_kernel<T, WM / 2, NC, FOLDS, ZEROS>(a, s);
    } else {
        static std::atomic<bool> set[64];
        auto kernel = gemm_w4_tile_kernel<T, WM, NC, FOLDS, ZEROS, 3>;
        if (hipError_t e = allow_lds(kernel, set)) return e;
        return launch_args(kernel, dim3((unsigned)(ceil_div(a.m, C::ROWS) * ceil_div(a.n, C::COLUMNS))), dim3(C::THREADS), C::LDS_BYTES, s, a);
    }
}

template <typename T, int WM, int NC>
hipError_t launch_tile(const GemmW4Args &a, hipStream_t s)
{
    auto folds = [&](auto n) {
        return a.w.zeros ? launch_tile_kernel<T, WM, NC, decltype(n)::value, true>(a, s) : launch_tile_kernel<T, WM, NC, decltype(n)::value, false>(a, s);
    };
    if (a.group % 128 == 0) return folds(std::integral_constant<int, 1>());
    if (a.group % 64 == 0) return folds(std::integral_constant<int, 2>());
    return folds(std::integral_constant<int, 4>());
}

// More than 32 columns: what a call takes by each kernel, in us, from rounds of work-groups over the 256 CUs.  Measured, fp16 and bf16, group 128:
//   stream, 32 x 32 (or 16 x 32): what a work-group pulls at some 47 bytes a ns    128 x 4096 x 4096 17.3, 256 30-32, 512 57-61; 64 x 8192 x 8192 29
//   tile of 64 x 64, two a CU: 1.1 us a slot of 128 places, 1.4 for a CU with two   256 x 8192 x 4096 45, 512 x 4096 x 4096 45, 1024 87
//   tile of 256 x 128: 2.1 us a slot                                               512 x 4096 x 4096 64, 1024 66, 2048 x 8192 x 4096 137 and 147
enum class Kernel { kStream16, kStream32, kTile64, kTile256 };
Kernel kernel_for(size_t m, size_t n, size_t k)
{
    const double slots = (double)ceil_div(k, 128);
    const size_t tiles32 = ceil_div(m, 32) * ceil_div(n, 32), tiles16 = ceil_div(m, 16) * ceil_div(n, 32), tiles64 = ceil_div(m, 64) * ceil_div(n, 64),
                 tiles256 = ceil_div(m, 256) * ceil_div(n, 128);
    const double us[4] = {(double)ceil_div(tiles16, 256) * (double)k * 72 / 47e3, (double)ceil_div(tiles32, 256) * (double)k * 80 / 47e3,
                          (tiles64 <= 256 ? 1.1 : 1.4 * (double)ceil_div(tiles64, 512)) * slots, 2.1 * (double)ceil_div(tiles256, 256) * slots};
    return (Kernel)(std::min_element(us, us + 4) - us);
}

template <typename T>
hipError_t launch_columns(const GemmW4Args &a, hipStream_t s)
{
    if (a.n == 1) return launch_stream_columns<T, 1>(a, s);
    if (a.n <= 4) return launch_stream_columns<T, 4>(a, s);
    if (a.n <= 16) return launch_stream_columns<T, 16>(a, s);
    if (a.n <= 32) return launch_stream_columns<T, 32>(a, s);
    switch (kernel_for(a.m, a.n, a.k)) {
        case Kernel::kStream16: return launch_stream_tile<T, 32, 1>(a, s);
        case Kernel::kStream32: return launch_stream_tile<T, 32, 2>(a, s);
        case Kernel::kTile64: return launch_tile<T, 2, 4>(a, s);
        default: return launch_tile<T, 8, 8>(a, s);
    }
}

template <typename T>
hipError_t launch_gemm(const GemmW4Args &all, hipStream_t s)
{
    // what one launch may be: a grid has less than 2^32 threads
    constexpr uint64_t kRows = 1u << 22, kColumns = 1u << 16;
    for (uint64_t i = 0; i < all.m; i += kRows)
        for (uint64_t j = 0; j < all.n; j += kColumns) {
            GemmW4Args a = all;
            a.m = (uint32_t)std::min(all.m - i, kRows);
            a.n = (uint32_t)std::min(all.n - j, kColumns);
            a.w.q += i * a.w.ldq;
            a.w.scales = static_cast<const T *>(a.w.scales) + i * a.w.lds;
            if (a.w.zeros) a.w.zeros += i * a.w.ldz;
            a.B = static_cast<const T *>(all.B) + j * all.ldb;
            a.C = static_cast<T *>(all.C) + i + j * all.ldc;
            if (hipError_t e = launch_columns<T>(a, s)) return e;
        }
    return hipSuccess;
}

}  // namespace
}  // namespace mmbo

using namespace mmbo;

extern "C" {

int mmbo_gemm_w4(int dtype, size_t m, size_t n, size_t k, size_t group, const void *alpha, const void *Q, size_t ldq,
                 const void *scales, size_t lds, const unsigned char *zeros, size_t ldz, const void *B, size_t ldb,
                 const void *beta, void *C, size_t ldc, void *stream)
{
    if (!w4_dtype(dtype)) return MMBO_ERR_INVALID_DTYPE;
    if (!alpha || !beta) return MMBO_ERR_NULL_POINTER;
    if (int rc = check_weight(m, k, group, ldq, lds, zeros, ldz)) return rc;
    if (n > kMaxDim || ldb > kMaxDim || ldc > kMaxDim) return MMBO_ERR_INVALID_SIZE;
    if (ldb < std::max<size_t>(k, 1) || ldc < std::max<size_t>(m, 1)) return MMBO_ERR_INVALID_SIZE;
    if (m == 0 || n == 0) return MMBO_OK;
    if (!C || (k != 0 && (!Q || !scales || !B))) return MMBO_ERR_NULL_POINTER;
    const GemmW4Args a{matrix_of(Q, ldq, scales, lds, zeros, ldz), B, C, *static_cast<const float *>(alpha), *static_cast<const float *>(beta),
                       (uint32_t)m, (uint32_t)n, (uint32_t)k, (uint32_t)group, ldb, ldc};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return status_of(dtype == MMBO_F16 ? launch_gemm<half_t>(a, s) : launch_gemm<bf16_t>(a, s));
}

// Not part of the interface: mmbo_gemm_w4 for packed operands by a given kernel -- 0, 1: 16 or 32 rows of 32 columns on the stream, 2, 3: tiles of 64 x 64 and
// 256 x 128 -- whatever the pick is: the tests reach each of them through it.
int mmbo_internal_gemm_w4(int kernel, int dtype, size_t m, size_t n, size_t k, size_t group, const void *Q, const void *scales, const unsigned char *zeros,
                          const void *B, void *C, void *stream)
{
    if (!w4_dtype(dtype)) return MMBO_ERR_INVALID_DTYPE;
    if (kernel < 0 || kernel > 3) return MMBO_ERR_INVALID_CONFIG;
    const size_t ldq = (k + 1) / 2 * 2, groups = ceil_div(k, std::max<size_t>(group, 1));
    if (int rc = check_weight(m, k, group, ldq, groups, zeros, groups)) return rc;
    if (m == 0 || n == 0 || k == 0 || m > 1 << 22 || n > 1 << 16) return MMBO_ERR_INVALID_SIZE;
    const GemmW4Args a{matrix_of(Q, ldq, scales, groups, zeros, groups), B, C, 1.0f, 0.0f, (uint32_t)m, (uint32_t)n, (uint32_t)k, (uint32_t)group, k, m};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return kernel == 0 ? launch_stream_tile<T, 32, 1>(a, s) : kernel == 1 ? launch_stream_tile<T, 32, 2>(a, s) : kernel == 2 ? launch_tile<T, 2, 4>(a, s) : launch_tile<T, 8, 8>(a, s);
    };
    return status_of(dtype == MMBO_F16 ? run((half_t *)nullptr) : run((bf16_t *)nullptr));
}

int mmbo_w4_quantize(int w_dtype, int dtype, size_t m, size_t k, size_t group, const void *W, size_t ldw, void *Q, size_t ldq,
                     void *scales, size_t lds, unsigned char *zeros, size_t ldz, void *stream)
{
    if (!w4_dtype(dtype) || !(w4_dtype(w_dtype) || w_dtype == MMBO_F32)) return MMBO_ERR_INVALID_DTYPE;
    if (int rc = check_weight(m, k, group, ldq, lds, zeros, ldz)) return rc;
    if (ldw > kMaxDim || ldw < k) return MMBO_ERR_INVALID_SIZE;
    if (m == 0 || k == 0) return MMBO_OK;
    if (!W || !Q || !scales) return MMBO_ERR_NULL_POINTER;
    const size_t groups = ceil_div(k, group);
    QuantArgs a{matrix_of(Q, ldq, scales, lds, zeros, ldz), const_cast<void *>(W), ldw, 0, (uint32_t)k, (uint32_t)group, (uint32_t)groups};
    hipStream_t s = static_cast<hipStream_t>(stream);
    // lanes for a group of any size: a power of two
    const size_t wsize = w_dtype == MMBO_F32 ? 4 : 2, most = ceil_div(std::min(group, k), kQuantElements);
    size_t lanes = 2;
    while (lanes < 64 && lanes < most) lanes *= 2;
    auto launch = [&](auto *w, auto *t) {
        using TW = std::remove_pointer_t<decltype(w)>;
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid((unsigned)ceil_div(a.m * groups * lanes, 256)), block(256);
        return lanes == 2    ? launch_args(w4_quantize_kernel<TW, T, 2>, grid, block, 0, s, a)
               : lanes == 4  ? launch_args(w4_quantize_kernel<TW, T, 4>, grid, block, 0, s, a)
               : lanes == 8  ? launch_args(w4_quantize_kernel<TW, T, 8>, grid, block, 0, s, a)
               : lanes == 16 ? launch_args(w4_quantize_kernel<TW, T, 16>, grid, block, 0, s, a)
               : lanes == 32 ? launch_args(w4_quantize_kernel<TW, T, 32>, grid, block, 0, s, a)
                             : launch_args(w4_quantize_kernel<TW, T, 64>, grid, block, 0, s, a);
    };
    auto by_weight = [&](auto *t) {
        return w_dtype == MMBO_F32 ? launch((float *)nullptr, t) : w_dtype == MMBO_F16 ? launch((half_t *)nullptr, t) : launch((bf16_t *)nullptr, t);
    };
    const size_t esz = 2;
    return by_rows(m, groups * lanes, [&](size_t i, size_t rows) {
        a.m = (uint32_t)rows;
        a.W = const_cast<char *>(static_cast<const char *>(W)) + i * ldw * wsize;
        a.w = matrix_of(static_cast<const char *>(Q) + i * (ldq / 2), ldq, static_cast<const char *>(scales) + i * lds * esz, lds, zeros ? zeros + i * ldz : nullptr, ldz);
        return dtype == MMBO_F16 ? by_weight((half_t *)nullptr) : by_weight((bf16_t *)nullptr);
    });
}

int mmbo_w4_dequantize(int dtype, size_t m, size_t k, size_t group, const void *Q, size_t ldq, const void *scales, size_t lds,
                       const unsigned char *zeros, size_t ldz, void *W, size_t ldw, void *stream)
{
    if (!w4_dtype(dtype)) return MMBO_ERR_INVALID_DTYPE;
    if (int rc = check_weight(m, k, group, ldq, lds, zeros, ldz)) return rc;
    if (ldw > kMaxDim || ldw < k) return MMBO_ERR_INVALID_SIZE;
    if (m == 0 || k == 0) return MMBO_OK;
    if (!W || !Q || !scales) return MMBO_ERR_NULL_POINTER;
    QuantArgs a{matrix_of(Q, ldq, scales, lds, zeros, ldz), W, ldw, 0, (uint32_t)k, (uint32_t)group, (uint32_t)ceil_div(k, group)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t threads = ceil_div(k, 32) * 4, esz = 2;
    return by_rows(m, threads, [&](size_t i, size_t rows) {
        a.m = (uint32_t)rows;
        a.W = static_cast<char *>(W) + i * ldw * esz;
        a.w = matrix_of(static_cast<const char *>(Q) + i * (ldq / 2), ldq, static_cast<const char *>(scales) + i * lds * esz, lds, zeros ? zeros + i * ldz : nullptr, ldz);
        const dim3 grid((unsigned)ceil_div(rows * threads, 256));
        return dtype == MMBO_F16 ? launch_args(w4_dequantize_kernel<half_t>, grid, dim3(256), 0, s, a)
                                 : launch_args(w4_dequantize_kernel<bf16_t>, grid, dim3(256), 0, s, a);
    });
}

}  // extern "C"
