// C ABI of the mixture-of-experts layer for a few tokens: argument checks, workspace, launches and kernels.
#include "../../include/mmbo_gemm.h"

#include <algorithm>

#include "w4.hpp"

namespace mmbo {
namespace {

struct MoeMatrix {
    W4Matrix w4;                                // 4-bit weights; of 16-bit ones w4.q is their address and w4.ldq their bytes from row to row
    int64_t stride, stride_scales, stride_zeros;    // bytes, groups, groups from expert to expert
};

struct MoeArgs {
    MoeMatrix gate_up, down;
    const void *router, *x;
    const float *bias;
    void *y;
    double *logits;                             // [tokens][experts]
    float *inner_values;                        // h: [tokens * top_k][inner]
    int *ids;                                   // [tokens][top_k]
    float *weights;
    float alpha, beta;
    uint32_t tokens, hidden, inner, experts, top_k, group;
    uint64_t ldx, ldy, ld_router;
    int sigmoid, renormalize;
};

// Element l of row i of a matrix that starts at (q, scales, zeros).
template <typename T, bool W4>
__device__ inline float weight(const MoeMatrix &m, uint32_t expert, uint64_t i, uint32_t l, uint32_t group)
{
    const uint8_t *q = m.w4.q + (int64_t)expert * m.stride + i * m.w4.ldq;
    if constexpr (!W4) return (float)reinterpret_cast<const T *>(q)[l];
    const uint32_t g = l / group;
    const float s = (float)static_cast<const T *>(m.w4.scales)[(int64_t)expert * m.stride_scales + g + i * m.w4.lds];
    const float z = m.w4.zeros ? (float)(m.w4.zeros[(int64_t)expert * m.stride_zeros + g + i * m.w4.ldz] & kW4ZeroMask) : kW4Zero;
    return ((float)(l & 1 ? q[l / 2] >> 4 : q[l / 2] & 15) - z) * s;
}

__device__ inline double wave_sum(double v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ inline float wave_sum(float v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// A wavefront: the logit of one expert for one token.
template <typename T, typename TR>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a)
{
    const uint32_t lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= a.tokens * a.experts) return;
    const uint32_t t = at / a.experts, e = at % a.experts;
    const T *x = static_cast<const T *>(a.x) + t * a.ldx;
    const TR *r = static_cast<const TR *>(a.router) + e * a.ld_router;
    double v = 0.0;
    for (uint32_t l = lane; l < a.hidden; l += 64) v = __builtin_fma((double)(float)r[l], (double)(float)x[l], v);
    v = wave_sum(v);
    if (lane == 0) a.logits[at] = v;
}

// A wavefront: the selection of one token.
__global__ void __launch_bounds__(64) moe_select_kernel(const MoeArgs a)
{
    __shared__ double keys[MMBO_MOE_MAX_EXPERTS];
    const uint32_t t = blockIdx.x, lane = threadIdx.x;
    const double *logits = a.logits + (uint64_t)t * a.experts;
    const double lowest = -__builtin_huge_val();
    double most = lowest, sum = 0.0;
    for (uint32_t e = lane; e < a.experts; e += 64) most = fmax(most, logits[e]);
    for (int d = 32; d > 0; d >>= 1) most = fmax(most, __shfl_xor(most, d));
    for (uint32_t e = lane; e < a.experts; e += 64) sum += exp(logits[e] - most);
    sum = wave_sum(sum);
    auto score = [&](uint32_t e) { return a.sigmoid ? 1.0 / (1.0 + exp(-logits[e])) : exp(logits[e] - most) / sum; };
    for (uint32_t e = lane; e < a.experts; e += 64) {
        const double key = a.bias ? score(e) + (double)a.bias[e] : logits[e];
        keys[e] = key != key ? lowest : key;
    }
    __syncthreads();
    uint64_t taken = 0;                         // of this lane's experts, lane + 64 * b: bit b
    double total = 0.0, mine = 0.0;
    int mine_id = 0;
    for (uint32_t s = 0; s < a.top_k; ++s) {
        double best = lowest;
        uint32_t id = 0xFFFFFFFFu;
        for (uint32_t e = lane, b = 0; e < a.experts; e += 64, ++b)
            if (!(taken >> b & 1) && (id == 0xFFFFFFFFu || keys[e] > best)) { best = keys[e]; id = e; }
        for (int d = 32; d > 0; d >>= 1) {
            const double other = __shfl_xor(best, d);
            const uint32_t oid = __shfl_xor(id, d);
            if (oid != 0xFFFFFFFFu && (id == 0xFFFFFFFFu || other > best || (other == best && oid < id))) { best = other; id = oid; }
        }
        if ((id & 63) == lane) taken |= 1ull << (id >> 6);
        const double v = score(id);
        total += v;
        if (lane == s) { mine = v; mine_id = (int)id; }
    }
    if (lane < a.top_k) {
        const double w = !a.renormalize ? mine : total == 0.0 ? 0.0 : mine / total;
        a.ids[(uint64_t)t * a.top_k + lane] = mine_id;
        a.weights[(uint64_t)t * a.top_k + lane] = (float)w;
    }
}

// A wavefront: one element of h of one token and one of its experts.
template <typename T, bool W4>
__global__ void __launch_bounds__(256) moe_gate_up_kernel(const MoeArgs a)
{
    const uint32_t lane = threadIdx.x & 63, i = blockIdx.x * 4 + (threadIdx.x >> 6), p = blockIdx.y;
    if (i >= a.inner) return;
    const uint32_t e = (uint32_t)a.ids[p];
    const T *x = static_cast<const T *>(a.x) + p / a.top_k * a.ldx;
    float g = 0.0f, u = 0.0f;
    for (uint32_t l = lane; l < a.hidden; l += 64) {
        const float v = (float)x[l];
        g = __builtin_fmaf(weight<T, W4>(a.gate_up, e, i, l, a.group), v, g);
        u = __builtin_fmaf(weight<T, W4>(a.gate_up, e, (uint64_t)a.inner + i, l, a.group), v, u);
    }
    g = wave_sum(g);
    u = wave_sum(u);
    if (lane == 0) a.inner_values[(uint64_t)p * a.inner + i] = g / (1.0f + expf(-g)) * u;
}

// A wavefront: one element of y.
template <typename T, bool W4>
__global__ void __launch_bounds__(256) moe_down_kernel(const MoeArgs a)
{
    const uint32_t lane = threadIdx.x & 63, i = blockIdx.x * 4 + (threadIdx.x >> 6), t = blockIdx.y;
    if (i >= a.hidden) return;
    float sum = 0.0f;
    for (uint32_t s = 0; s < a.top_k; ++s) {
        const uint64_t p = (uint64_t)t * a.top_k + s;
        const uint32_t e = (uint32_t)a.ids[p];
        float v = 0.0f;
        for (uint32_t l = lane; l < a.inner; l += 64) v = __builtin_fmaf(weight<T, W4>(a.down, e, i, l, a.group), a.inner_values[p * a.inner + l], v);
        sum = __builtin_fmaf(a.weights[p], wave_sum(v), sum);
    }
    if (lane == 0) {
        T *y = static_cast<T *>(a.y) + t * a.ldy + i;
        float v = a.alpha * sum;
        if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*y, v);
        *y = (T)v;
    }
}

constexpr size_t kMaxDim = 0x7FFFFFFFull;

int check_matrix(const mmbo_moe_matrix &w, size_t k, size_t group)
{
    if (w.ld > kMaxDim || w.ld < k || w.stride < 0) return MMBO_ERR_INVALID_SIZE;
    if (group != 0) {
        const size_t groups = (k + group - 1) / group;
        if (w.ld % 2 != 0 || w.stride % 2 != 0 || w.lds > kMaxDim || w.lds < groups || w.stride_scales < 0) return MMBO_ERR_INVALID_SIZE;
        if (w.zeros && (w.ldz > kMaxDim || w.ldz < groups || w.stride_zeros < 0)) return MMBO_ERR_INVALID_SIZE;
    }
    return MMBO_OK;
}

int check_layer(const mmbo_moe_layer *l)
{
    if (!l) return MMBO_ERR_NULL_POINTER;
    if (!w4_dtype(l->dtype) || (l->router_dtype != l->dtype && l->router_dtype != MMBO_F32)) return MMBO_ERR_INVALID_DTYPE;
    if (l->scoring != MMBO_MOE_SOFTMAX && l->scoring != MMBO_MOE_SIGMOID) return MMBO_ERR_INVALID_OP;
    if (l->hidden == 0 || l->hidden > kMaxDim || l->inner == 0 || l->inner > kMaxDim / 2) return MMBO_ERR_INVALID_SIZE;
    if (l->experts == 0 || l->experts > MMBO_MOE_MAX_EXPERTS || l->top_k == 0 || l->top_k > MMBO_MOE_MAX_TOP_K || l->top_k > l->experts)
        return MMBO_ERR_INVALID_SIZE;
    if (l->group % kW4Group != 0 || l->group > kMaxDim || l->ld_router > kMaxDim || l->ld_router < l->hidden) return MMBO_ERR_INVALID_SIZE;
    if (int rc = check_matrix(l->gate_up, l->hidden, l->group)) return rc;
    return check_matrix(l->down, l->inner, l->group);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// Places of the workspace's parts, in bytes.
struct Parts {
    size_t logits, inner_values, ids, weights, all;
};
Parts parts_of(const mmbo_moe_layer &l, size_t tokens)
{
    Parts p;
    p.logits = 0;
    p.inner_values = p.logits + round16(tokens * l.experts * sizeof(double));
    p.ids = p.inner_values + round16(tokens * l.top_k * l.inner * sizeof(float));
    p.weights = p.ids + round16(tokens * l.top_k * sizeof(int));
    p.all = p.weights + round16(tokens * l.top_k * sizeof(float));
    return p;
}

MoeMatrix matrix_of(const mmbo_moe_matrix &w, bool w4)
{
    MoeMatrix m{};
    m.w4.q = static_cast<const uint8_t *>(w.data);
    m.w4.ldq = w4 ? w.ld / 2 : w.ld * 2;
    m.stride = w4 ? w.stride / 2 : w.stride * 2;
    if (w4) {
        m.w4.scales = w.scales; m.w4.lds = w.lds; m.stride_scales = w.stride_scales;
        m.w4.zeros = w.zeros; m.w4.ldz = w.ldz; m.stride_zeros = w.stride_zeros;
    }
    return m;
}

template <typename T>
hipError_t run(const MoeArgs &a, bool router32, hipStream_t s)
{
    const dim3 block(256);
    const unsigned logits = (a.tokens * a.experts + 3) / 4;
    hipError_t e = router32 ? launch_args(moe_logits_kernel<T, float>, dim3(logits), block, 0, s, a)
                            : launch_args(moe_logits_kernel<T, T>, dim3(logits), block, 0, s, a);
    if (e != hipSuccess) return e;
    e = launch_args(moe_select_kernel, dim3(a.tokens), dim3(64), 0, s, a);
    if (e != hipSuccess) return e;
    const dim3 up((a.inner + 3) / 4, a.tokens * a.top_k), down((a.hidden + 3) / 4, a.tokens);
    e = a.group ? launch_args(moe_gate_up_kernel<T, true>, up, block, 0, s, a) : launch_args(moe_gate_up_kernel<T, false>, up, block, 0, s, a);
    if (e != hipSuccess) return e;
    return a.group ? launch_args(moe_down_kernel<T, true>, down, block, 0, s, a) : launch_args(moe_down_kernel<T, false>, down, block, 0, s, a);
}

}  // namespace
}  // namespace mmbo

using namespace mmbo;

extern "C" {

size_t mmbo_moe_workspace_bytes(const mmbo_moe_layer *layer, size_t tokens)
{
    if (check_layer(layer) != MMBO_OK || tokens > MMBO_MOE_MAX_TOKENS) return 0;
    return std::max<size_t>(parts_of(*layer, tokens).all, 16);
}

int mmbo_moe(const mmbo_moe_layer *layer, size_t tokens, const void *alpha, const void *x, size_t ldx, const void *beta, void *y,
             size_t ldy, int *ids, float *weights, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_layer(layer)) return rc;
    const mmbo_moe_layer &l = *layer;
    if (!alpha || !beta) return MMBO_ERR_NULL_POINTER;
    if (tokens > MMBO_MOE_MAX_TOKENS || ldx > kMaxDim || ldy > kMaxDim || ldx < l.hidden || ldy < l.hidden) return MMBO_ERR_INVALID_SIZE;
    if (tokens == 0) return MMBO_OK;
    if (!x || !y || !workspace || !l.router || !l.gate_up.data || !l.down.data) return MMBO_ERR_NULL_POINTER;
    if (l.group && (!l.gate_up.scales || !l.down.scales)) return MMBO_ERR_NULL_POINTER;
    const Parts p = parts_of(l, tokens);
    if (workspace_bytes < p.all || (uintptr_t)workspace % 16 != 0) return MMBO_ERR_WORKSPACE;
    char *ws = static_cast<char *>(workspace);
    MoeArgs a{};
    a.gate_up = matrix_of(l.gate_up, l.group != 0);
    a.down = matrix_of(l.down, l.group != 0);
    a.router = l.router; a.ld_router = l.ld_router; a.bias = l.bias;
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy;
    a.alpha = *static_cast<const float *>(alpha); a.beta = *static_cast<const float *>(beta);
    a.logits = reinterpret_cast<double *>(ws + p.logits);
    a.inner_values = reinterpret_cast<float *>(ws + p.inner_values);
    a.ids = ids ? ids : reinterpret_cast<int *>(ws + p.ids);
    a.weights = weights ? weights : reinterpret_cast<float *>(ws + p.weights);
    a.tokens = (uint32_t)tokens; a.hidden = (uint32_t)l.hidden; a.inner = (uint32_t)l.inner; a.experts = (uint32_t)l.experts;
    a.top_k = (uint32_t)l.top_k; a.group = (uint32_t)l.group;
    a.sigmoid = l.scoring == MMBO_MOE_SIGMOID; a.renormalize = l.renormalize != 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool router32 = l.router_dtype == MMBO_F32;
    const hipError_t e = l.dtype == MMBO_F16 ? run<half_t>(a, router32, s) : run<bf16_t>(a, router32, s);
    return e == hipSuccess ? MMBO_OK : report_hip_error(e);
}

}  // extern "C"
