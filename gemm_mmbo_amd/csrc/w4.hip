// C ABI of the products with 4-bit weights and of their format: argument checks and dispatch; quantize and dequantize.
#include "../../include/mmbo_gemm.h"

#include <algorithm>

#include "w4.hpp"

namespace mmbo {
namespace {

template <typename T>
__device__ inline float load_scale(const void *p, uint64_t at) { return (float)static_cast<const T *>(p)[at]; }

// A wavefront has one row of W and up to four columns of B; its lanes share k, eight places of a dword of codes at a time.
template <typename T>
__global__ void __launch_bounds__(256) gemm_w4_rows_kernel(const GemmW4Args a)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t i = (uint64_t)blockIdx.x * 4 + wave;
    if (i >= a.m) return;
    for (uint64_t j0 = (uint64_t)blockIdx.y * 4; j0 < a.n; j0 += (uint64_t)gridDim.y * 4) {
        float acc[4] = {};
        for (uint64_t l0 = lane * 8; l0 < a.k; l0 += 512) {
            const uint32_t g = (uint32_t)(l0 / a.group);
            const float s = load_scale<T>(a.w.scales, g + i * a.w.lds);
            const float z = a.w.zeros ? (float)a.w.zeros[g + i * a.w.ldz] : kW4Zero;
            for (uint32_t e = 0; e < 8 && l0 + e < a.k; ++e) {
                const uint64_t l = l0 + e;
                const uint8_t byte = a.w.q[i * a.w.ldq + l / 2];
                const float w = ((float)(l & 1 ? byte >> 4 : byte & 15) - z) * s;
                for (uint32_t j = 0; j < 4; ++j)
                    if (j0 + j < a.n) acc[j] = __builtin_fmaf(w, (float)static_cast<const T *>(a.B)[l + (j0 + j) * a.ldb], acc[j]);
            }
        }
        for (uint32_t j = 0; j < 4; ++j) {
            float v = acc[j];
            for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
            if (lane == 0 && j0 + j < a.n) {
                T *c = static_cast<T *>(a.C) + i + (j0 + j) * a.ldc;
                v *= a.alpha;
                if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*c, v);
                *c = (T)v;
            }
        }
    }
}

template <typename T> struct Limits;
template <> struct Limits<float> { static constexpr float largest = 3.40282346638528859812e38f; };
template <> struct Limits<half_t> { static constexpr float largest = 65504.0f; };
template <> struct Limits<bf16_t> { static constexpr float largest = 3.38953138925153547590e38f; };

// w as the format counts it: NaN is 0, an infinity the largest finite number
template <typename TW>
__device__ inline float finite(float w)
{
    const float most = Limits<TW>::largest;
    return w != w ? 0.0f : fminf(fmaxf(w, -most), most);
}

// The whole number nearest to w / s, halves to even, for numbers within 16 or clamped there: the quotient's rounding may pick the wrong one next to
// a border, and the remainder w - n * s, which is exact in fp32, says so.
__device__ inline float nearest(float w, float s)
{
    float n = rintf(fminf(fmaxf(w / s, -16.0f), 16.0f));
    const float r = __builtin_fmaf(-n, s, w), half = 0.5f * s;
    const bool odd = ((int)n & 1) != 0;
    if (r > half || (r == half && odd)) n += 1.0f;
    else if (r < -half || (r == -half && odd)) n -= 1.0f;
    return n;
}

// One thread: one group of one row.
template <typename TW, typename T>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const QuantArgs a)
{
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (uint64_t)a.m * a.groups) return;
    const uint64_t i = at / a.groups;
    const uint32_t g = (uint32_t)(at % a.groups);
    const uint64_t l0 = (uint64_t)g * a.group, l1 = l0 + a.group < a.k ? l0 + a.group : a.k;
    const TW *w = static_cast<const TW *>(a.W) + i * a.ldw;
    float low = 0.0f, high = 0.0f;
    for (uint64_t l = l0; l < l1; ++l) {
        const float v = finite<TW>((float)w[l]);
        low = fminf(low, v);
        high = fmaxf(high, v);
    }
    const bool zeros = a.w.zeros != nullptr;
    // (in 64 bits: high - low may pass the largest float)
    float s = zeros ? (float)(((double)high - (double)low) / 15.0) : fmaxf(high, -low) / 7.0f;
    s = (float)(T)fminf(s, Limits<T>::largest);
    float z = zeros ? 0.0f : kW4Zero;
    if (zeros && s != 0.0f) z = fminf(fmaxf(nearest(-low, s), 0.0f), 15.0f);
    static_cast<T *>(const_cast<void *>(a.w.scales))[g + i * a.w.lds] = (T)s;
    if (zeros) const_cast<uint8_t *>(a.w.zeros)[g + i * a.w.ldz] = (uint8_t)z;
    uint8_t *q = const_cast<uint8_t *>(a.w.q) + i * a.w.ldq;
    for (uint64_t l = l0; l < l1; l += 2) {
        uint32_t code[2] = {0, 0};
        for (int e = 0; e < 2; ++e)
            if (l + e < l1) code[e] = (uint32_t)(s == 0.0f ? z : fminf(fmaxf(nearest(finite<TW>((float)w[l + e]), s) + z, 0.0f), 15.0f));
        q[l / 2] = (uint8_t)(code[0] | code[1] << 4);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const QuantArgs a)
{
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (uint64_t)a.m * a.k) return;
    const uint64_t i = at / a.k, l = at % a.k;
    const uint32_t g = (uint32_t)(l / a.group);
    const uint8_t byte = a.w.q[i * a.w.ldq + l / 2];
    const float z = a.w.zeros ? (float)a.w.zeros[g + i * a.w.ldz] : kW4Zero;
    static_cast<T *>(a.W)[i * a.ldw + l] = (T)(((float)(l & 1 ? byte >> 4 : byte & 15) - z) * load_scale<T>(a.w.scales, g + i * a.w.lds));
}

constexpr size_t kMaxDim = 0x7FFFFFFFull;

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
    const dim3 grid((unsigned)((m + 3) / 4), (unsigned)std::min<size_t>((n + 3) / 4, 65535));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return status_of(dtype == MMBO_F16 ? launch_args(gemm_w4_rows_kernel<half_t>, grid, dim3(256), 0, s, a)
                                       : launch_args(gemm_w4_rows_kernel<bf16_t>, grid, dim3(256), 0, s, a));
}

int mmbo_w4_quantize(int w_dtype, int dtype, size_t m, size_t k, size_t group, const void *W, size_t ldw, void *Q, size_t ldq,
                     void *scales, size_t lds, unsigned char *zeros, size_t ldz, void *stream)
{
    if (!w4_dtype(dtype) || !(w4_dtype(w_dtype) || w_dtype == MMBO_F32)) return MMBO_ERR_INVALID_DTYPE;
    if (int rc = check_weight(m, k, group, ldq, lds, zeros, ldz)) return rc;
    if (ldw > kMaxDim || ldw < k) return MMBO_ERR_INVALID_SIZE;
    if (m == 0 || k == 0) return MMBO_OK;
    if (!W || !Q || !scales) return MMBO_ERR_NULL_POINTER;
    const size_t groups = (k + group - 1) / group, blocks = (m * groups + 255) / 256;
    if (blocks > kMaxDim) return MMBO_ERR_INVALID_SIZE;
    const QuantArgs a{matrix_of(Q, ldq, scales, lds, zeros, ldz), const_cast<void *>(W), ldw, (uint32_t)m, (uint32_t)k, (uint32_t)group, (uint32_t)groups};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto *w, auto *t) {
        using TW = std::remove_pointer_t<decltype(w)>;
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_args(w4_quantize_kernel<TW, T>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    };
    auto by_weight = [&](auto *t) {
        return w_dtype == MMBO_F32 ? launch((float *)nullptr, t) : w_dtype == MMBO_F16 ? launch((half_t *)nullptr, t) : launch((bf16_t *)nullptr, t);
    };
    return status_of(dtype == MMBO_F16 ? by_weight((half_t *)nullptr) : by_weight((bf16_t *)nullptr));
}

int mmbo_w4_dequantize(int dtype, size_t m, size_t k, size_t group, const void *Q, size_t ldq, const void *scales, size_t lds,
                       const unsigned char *zeros, size_t ldz, void *W, size_t ldw, void *stream)
{
    if (!w4_dtype(dtype)) return MMBO_ERR_INVALID_DTYPE;
    if (int rc = check_weight(m, k, group, ldq, lds, zeros, ldz)) return rc;
    if (ldw > kMaxDim || ldw < k) return MMBO_ERR_INVALID_SIZE;
    if (m == 0 || k == 0) return MMBO_OK;
    if (!W || !Q || !scales) return MMBO_ERR_NULL_POINTER;
    const size_t blocks = (m * k + 255) / 256;
    if (blocks > kMaxDim) return MMBO_ERR_INVALID_SIZE;
    const QuantArgs a{matrix_of(Q, ldq, scales, lds, zeros, ldz), W, ldw, (uint32_t)m, (uint32_t)k, (uint32_t)group, (uint32_t)((k + group - 1) / group)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return status_of(dtype == MMBO_F16 ? launch_args(w4_dequantize_kernel<half_t>, dim3((unsigned)blocks), dim3(256), 0, s, a)
                                       : launch_args(w4_dequantize_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, s, a));
}

}  // extern "C"
