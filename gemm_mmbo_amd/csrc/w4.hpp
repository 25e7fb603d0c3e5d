// Weights in 4 bits with a scale and a zero point for each group of k: the format, and what its kernels share.
// (l, i): place l of k of row i.  Code (l, i) is half of byte (l + i * ldq) / 2, the low half for even l.
#pragma once

#include <atomic>

#include "launch.hpp"

namespace mmbo {

typedef __bf16 bf16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kW4Group = 32;               // groups are whole multiples of this
constexpr float kW4Zero = 8.0f;                 // the zero point where none is stored
constexpr uint8_t kW4ZeroMask = 127;            // what counts of a stored one: 128 + zero point has to be a bf16 number

// A weight as the kernels take it.
struct W4Matrix {
    const uint8_t *q;
    const void *scales;
    const uint8_t *zeros;                       // or null
    uint64_t ldq;                               // bytes from row to row
    uint64_t lds, ldz;                          // groups from row to row
};

struct GemmW4Args {
    W4Matrix w;
    const void *B;
    void *C;
    float alpha, beta;
    uint32_t m, n, k, group;
    uint64_t ldb, ldc;
};

struct QuantArgs {
    W4Matrix w;                                 // (written by quantize)
    void *W;                                    // (written by dequantize)
    uint64_t ldw;
    uint32_t m, k, group, groups;
};

constexpr size_t kMaxDim = 0x7FFFFFFFull;
constexpr unsigned kLds = 160 * 1024;           // of a CU

template <typename N>
constexpr size_t ceil_div(size_t n, N by) { return (n + by - 1) / by; }

inline bool w4_dtype(int dtype) { return dtype == 1 || dtype == 3; }             // MMBO_F16, MMBO_BF16

template <typename Args, typename Kernel>
inline hipError_t launch_args(Kernel kernel, dim3 grid, dim3 block, unsigned lds_bytes, hipStream_t stream, const Args &args)
{
    void *kargs[] = {const_cast<Args *>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, kargs, lds_bytes, stream);
}

// All of a CU's LDS to a kernel, asked for once a device.
template <typename Kernel>
hipError_t allow_lds(Kernel kernel, std::atomic<bool> (&set)[64])
{
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || (dev >= 0 && dev < 64 && set[dev].load(std::memory_order_acquire))) return e;
    e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e == hipSuccess && dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
    return e;
}

}  // namespace mmbo
