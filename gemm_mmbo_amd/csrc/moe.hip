// C ABI of the mixture-of-experts layer for a few tokens: argument checks, workspace, launches and kernels.
#include "../../include/mmbo_gemm.h"

#include <algorithm>
#include <type_traits>

#include "stream.hpp"

namespace mmbo {
namespace {

constexpr uint32_t kTokens = 64;                // worked on at a time: a row of the grids

// h between the two products is fp32, in bf16 numbers that add up to it: 8 of its 24 bits each, with its range (two numbers of the layer's type held 16 bits in bf16,
// and in fp16 nothing above 65504 and less and less below 2^-13).  They lie in three planes; for 16 columns of 16-bit weights it lies as it is (kWhole), eight places at a time, four
// of them in the first plane and four in the second, and is taken apart behind LDS.
// A third less comes through a CU that way, for 44 vector instructions to 32 places, which 16 rows of 16-bit weights leave room for and 4-bit ones do not: 512 tokens, 8 of 64 experts of
// 2048 x 1024 1,133 us, in planes 1,236; 64 tokens, 2 of 16 experts of 4096 x 2048 in 4 bits 115 us, in planes 101.
constexpr int kPlanes = 3;
template <bool W4, int N2> constexpr bool kWhole = N2 > 4 && !W4;

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
    bf16_t *h;                                  // [plane][tokens * top_k][ld_h]
    char *table;                                // of each row of tokens
    float *parts;                               // sums of work-groups that share a tile of y: [row of tokens][tile][sharer][token][element]
    uint32_t *arrived;                          // how many of them are done: [row of tokens][tile]
    uint32_t *chosen;                           // the selection: [tokens][top_k]
    float *chosen_weights;
    uint32_t *selected;                         // work-groups of a row that have selected
    int *ids;                                   // [tokens][top_k]; either may be null
    float *weights;
    float alpha, beta;
    uint32_t tokens, hidden, inner, experts, top_k, group;
    uint32_t ld_h, columns, most_jobs, down_tiles, sharers;
    uint64_t ldx, ldy, ld_router;
    int sigmoid, renormalize;
};

__device__ inline double wave_sum(double v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Eight elements from `p`, of which `here` exist, as floats; the others are 0.
template <typename T>
__device__ inline void load8f(float (&v)[8], const T *p, int64_t here)
{
    if constexpr (sizeof(T) == 2) {
        const typename stream::Type<T>::Frag x = stream::frag_of<T>(stream::load8(p, here));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < here ? p[i] : 0.0f;
    }
}

// A work-group: the logits of one expert for up to kLogitTokens tokens.  The products of 16-bit numbers (and a router in fp32 by them) are summed in
// fp64: at 2^-53 a step, two experts change places where their logits differ by less than 1e-12 of what is summed.
// Bound by a launch and one round trip to memory: 4.4 us for 8 tokens of 2048 and 64 experts.
constexpr uint32_t kLogitTokens = 4;
template <typename T, typename TR>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a)
{
    __shared__ double parts[4][kLogitTokens];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x, t0 = blockIdx.y * kLogitTokens;
    if (e == 0 && t0 % kTokens == 0 && threadIdx.x == 0) a.selected[t0 / kTokens] = 0;
    const uint32_t count = min(kLogitTokens, a.tokens - t0);
    const TR *r = static_cast<const TR *>(a.router) + e * a.ld_router;
    const T *x = static_cast<const T *>(a.x) + t0 * a.ldx;
    double sums[kLogitTokens] = {};
    for (uint32_t l = threadIdx.x * 8; l < a.hidden; l += 2048) {
        float rv[8], xv[kLogitTokens][8];
        load8f(rv, r + l, (int64_t)a.hidden - l);
#pragma unroll
        for (uint32_t t = 0; t < kLogitTokens; ++t) load8f(xv[t], x + min(t, count - 1) * a.ldx + l, (int64_t)a.hidden - l);
#pragma unroll
        for (uint32_t t = 0; t < kLogitTokens; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[t] = __builtin_fma((double)rv[i], (double)xv[t][i], sums[t]);
    }
#pragma unroll
    for (uint32_t t = 0; t < kLogitTokens; ++t) {
        const double v = wave_sum(sums[t]);
        if (lane == 0) parts[wave][t] = v;
    }
    __syncthreads();
    if (threadIdx.x < count)
        a.logits[(uint64_t)(t0 + threadIdx.x) * a.experts + e] = parts[0][threadIdx.x] + parts[1][threadIdx.x] + parts[2][threadIdx.x] + parts[3][threadIdx.x];
}

// The (token, slot) pairs of a row of tokens by expert, and each expert's pairs in jobs of up to `columns`.
struct Table {
    uint32_t *count;                            // of jobs
    float *weight;                              // of a pair
    uint16_t *pair;                             // token of the row * top_k + slot: by expert, in order
    uint16_t *expert, *first;                   // of a job: its expert, and the place of its first pair; first[count] is where they end
};
__host__ __device__ inline uint32_t table_bytes(uint32_t pairs, uint32_t most_jobs) { return (16 + 6 * pairs + 4 * most_jobs + 2 + 15) / 16 * 16; }
__host__ __device__ inline Table table_at(char *at, uint32_t pairs, uint32_t most_jobs)
{
    Table t;
    t.count = reinterpret_cast<uint32_t *>(at);
    t.weight = reinterpret_cast<float *>(at + 16);
    t.pair = reinterpret_cast<uint16_t *>(t.weight + pairs);
    t.expert = t.pair + pairs;
    t.first = t.expert + most_jobs;
    return t;
}

// A number that orders as keys do, NaN below everything.
__device__ inline uint64_t order_of(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v != v ? 0 : b >> 63 ? ~b : b | 1ull << 63;
}
template <int CTRL>
__device__ inline uint64_t dpp64(uint64_t v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(v >> 32), CTRL, 0xf, 0xf, true);
    return (uint64_t)hi << 32 | lo;
}
// The largest of a wavefront's numbers, in every lane.
__device__ inline uint64_t wave_max(uint64_t v)
{
    v = max(v, dpp64<0x121>(v));                // rotations by 1, 2, 4, 8 within rows of 16
    v = max(v, dpp64<0x122>(v));
    v = max(v, dpp64<0x124>(v));
    v = max(v, dpp64<0x128>(v));
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    auto l16 = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), h16 = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = max((uint64_t)h16[0] << 32 | l16[0], (uint64_t)h16[1] << 32 | l16[1]);
    const uint32_t lo2 = (uint32_t)v, hi2 = (uint32_t)(v >> 32);
    auto l32 = __builtin_amdgcn_permlane32_swap(lo2, lo2, false, false), h32 = __builtin_amdgcn_permlane32_swap(hi2, hi2, false, false);
    return max((uint64_t)h32[0] << 32 | l32[0], (uint64_t)h32[1] << 32 | l32[1]);
}

// The selection of one token by a wavefront: lane s gets the expert of slot s and its weight.  PER: experts a lane has, lane + 64 * b.
template <int PER>
__device__ inline void select_token(const MoeArgs &a, uint32_t token, uint32_t lane, uint32_t &expert, float &weight)
{
    const double *logits = a.logits + (uint64_t)token * a.experts;
    double logit[PER];
    uint64_t key[PER];
    uint64_t most = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const uint32_t e = lane + 64 * b;
        logit[b] = e < a.experts ? logits[e] : -__builtin_huge_val();
        key[b] = e < a.experts ? order_of(logit[b]) : 0;
        most = max(most, key[b]);
    }
    // (One exp for all cases: on a CU that runs this once, time goes into fetching instructions.  A NaN among the logits is no largest one; it makes the
    // sum NaN, which scores that only count against each other do not need.)
    const bool over_sum = !a.sigmoid && (!a.renormalize || a.bias);
    if (!a.sigmoid) most = wave_max(most);
    const double highest = __builtin_bit_cast(double, most >> 63 ? most & ~(1ull << 63) : ~most);
    double score[PER], sum = 0.0;
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        const double v = exp(a.sigmoid ? -logit[b] : logit[b] - highest);
        score[b] = a.sigmoid ? 1.0 / (1.0 + v) : v;
        if (lane + 64 * b < a.experts) sum += v;
    }
    if (over_sum) {
        sum = 1.0 / wave_sum(sum);
#pragma unroll
        for (int b = 0; b < PER; ++b) score[b] *= sum;
    }
    if (a.bias)
#pragma unroll
        for (int b = 0; b < PER; ++b)
            if (lane + 64 * b < a.experts) key[b] = order_of(score[b] + (double)a.bias[lane + 64 * b]);
    uint32_t mine = 0, here = 0;             // the expert of slot `lane`; of this lane's experts, those that may still be taken
    double mine_score = 0.0;
#pragma unroll
    for (int b = 0; b < PER; ++b)
        if (lane + 64 * b < a.experts) here |= 1u << b;
    for (uint32_t s = 0; s < a.top_k; ++s) {
        uint64_t best = 0;
#pragma unroll
        for (int b = 0; b < PER; ++b)
            if (here >> b & 1) best = max(best, key[b]);
        best = wave_max(best);
        uint32_t e = 0;
        double v = 0.0;
        bool found = false;
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            const uint64_t who = __ballot((here >> b & 1) && key[b] == best);
            if (!found && who != 0) {
                const int l = __builtin_ctzll(who);
                const uint64_t bits = __builtin_bit_cast(uint64_t, score[b]);
                e = 64 * b + l;
                v = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(bits >> 32), l) << 32 |
                                                   (uint32_t)__builtin_amdgcn_readlane((uint32_t)bits, l));
                found = true;
            }
        }
        if (lane == (e & 63)) here &= ~(1u << (e >> 6));
        if (lane == s) {
            mine = e;
            mine_score = v;
        }
    }
    double v = mine_score;
    if (a.renormalize) {
        const double total = wave_sum(v);
        v = total == 0.0 ? 0.0 : v / total;
    }
    expert = mine;
    weight = (float)v;
}
__device__ inline void select_token(const MoeArgs &a, uint32_t token, uint32_t lane, uint32_t &expert, float &weight)
{
    if (a.experts <= 64) select_token<1>(a, token, lane, expert, weight);
    else if (a.experts <= 128) select_token<2>(a, token, lane, expert, weight);
    else select_token<8>(a, token, lane, expert, weight);
}

// A row's selection in LDS, and what a work-group needs to make its table.
struct Selection {
    uint16_t *id;                               // of a pair; whole eights of them
    uint16_t *before;                           // of a part of the pairs, for an expert: pairs by expert in front of it; whole eights
    uint16_t *jobs_before;                      // of an expert; whole eights
    float *weight;
    uint16_t *pair;                             // pairs by expert
};
constexpr uint32_t kMostParts = 512;            // (no work-group has more threads)
__host__ __device__ inline uint32_t eights(uint32_t n) { return (n + 7) / 8 * 8; }
__host__ __device__ inline uint32_t select_bytes(uint32_t pairs, uint32_t experts)
{
    return ((eights(pairs) + kMostParts + eights(experts)) * 2 + pairs * 6 + 15) / 16 * 16;
}
__device__ inline Selection selection_at(char *lds, uint32_t most_pairs, uint32_t experts)
{
    Selection s;
    s.id = reinterpret_cast<uint16_t *>(lds);
    s.before = s.id + eights(most_pairs);
    s.jobs_before = s.before + kMostParts;
    s.weight = reinterpret_cast<float *>(s.jobs_before + eights(experts));
    s.pair = reinterpret_cast<uint16_t *>(s.weight + most_pairs);
    return s;
}

// Sums of those in front of each of n <= 512 numbers (their sum stays below 2^16), by one wavefront, eight to a lane; their sum.  v: whole eights, aligned to them.
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
__device__ inline uint32_t scan(uint16_t *v, uint32_t n, uint32_t lane)
{
    u16x8 *const mine = reinterpret_cast<u16x8 *>(v) + lane;
    uint32_t own[8] = {}, sum = 0;
    if (lane * 8 < n) {
        const u16x8 q = *mine;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            own[i] = sum;
            if (lane * 8 + i < n) sum += q[i];
        }
    }
    uint32_t all = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t other = __shfl_up(all, d);
        if ((int)lane >= d) all += other;
    }
    if (lane * 8 < n) {
        u16x8 q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = (uint16_t)(all - sum + own[i]);
        *mine = q;
    }
    return __builtin_amdgcn_readlane(all, 63);
}

// The table of `pairs` pairs, by a work-group that has them in LDS.  A thread looks through a part of the pairs for an expert's, eight ids at a time: one thread
// to an expert, and a store to memory a pair, was 12 us for 128 pairs.
__device__ inline void make_table(const MoeArgs &a, uint32_t pairs, const Selection &sel, const Table &table)
{
    const u16x8 *const id8 = reinterpret_cast<const u16x8 *>(sel.id);
    const uint32_t pieces = (pairs + 7) / 8, parts = max(min(blockDim.x / a.experts, pieces), 1u);
    if (threadIdx.x < pieces * 8 - pairs) sel.id[pairs + threadIdx.x] = 0xFFFF;
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < a.experts * parts; x += blockDim.x) {
        const uint32_t e = x / parts, part = x % parts;
        uint32_t n = 0;
        for (uint32_t q = pieces * part / parts; q < pieces * (part + 1) / parts; ++q) {
            const u16x8 v = id8[q];
#pragma unroll
            for (int i = 0; i < 8; ++i) n += v[i] == e;
        }
        sel.before[x] = (uint16_t)n;
    }
    __syncthreads();
    if (threadIdx.x < 64) scan(sel.before, a.experts * parts, threadIdx.x);
    __syncthreads();
    auto end_of = [&](uint32_t e) { return e + 1 < a.experts ? (uint32_t)sel.before[(e + 1) * parts] : pairs; };
    for (uint32_t x = threadIdx.x; x < a.experts * parts; x += blockDim.x) {
        const uint32_t e = x / parts, part = x % parts;
        if (part == 0) sel.jobs_before[e] = (uint16_t)((end_of(e) - sel.before[x] + a.columns - 1) / a.columns);
        uint32_t at = sel.before[x];
        if (at == (x + 1 < a.experts * parts ? (uint32_t)sel.before[x + 1] : pairs)) continue;
        for (uint32_t q = pieces * part / parts; q < pieces * (part + 1) / parts; ++q) {
            const u16x8 v = id8[q];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (v[i] == e) sel.pair[at++] = (uint16_t)(q * 8 + i);
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t jobs = scan(sel.jobs_before, a.experts, threadIdx.x);
        if (threadIdx.x == 0) {
            *table.count = jobs;
            table.first[jobs] = (uint16_t)pairs;
        }
    }
    for (uint32_t i = threadIdx.x; i < pairs; i += blockDim.x) {
        const uint32_t p = sel.pair[i];
        table.pair[i] = (uint16_t)p;
        table.weight[i] = sel.weight[p];
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const uint32_t from = sel.before[e * parts], to = end_of(e);
        uint32_t job = sel.jobs_before[e];
        for (uint32_t n = from; n < to; n += a.columns, ++job) {
            table.expert[job] = (uint16_t)e;
            table.first[job] = (uint16_t)n;
        }
    }
}

__device__ inline char *table_of_row(const MoeArgs &a, uint32_t row) { return a.table + (uint64_t)row * table_bytes(min(kTokens, a.tokens) * a.top_k, a.most_jobs); }

// A wavefront: the selection of one token.  The work-group of a row that is done last makes the row's table (the counter was cleared by the kernel before).
constexpr uint32_t kSelectTokens = 4;           // of a work-group
__global__ void __launch_bounds__(kSelectTokens * 64) moe_select_kernel(const MoeArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ bool last;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.y;
    const uint32_t token0 = row * kTokens, tokens = min(kTokens, a.tokens - token0), pairs = tokens * a.top_k, most_pairs = min(kTokens, a.tokens) * a.top_k;
    const uint32_t t = blockIdx.x * kSelectTokens + wave;
    if (t < tokens) {
        uint32_t expert;
        float weight;
        select_token(a, token0 + t, lane, expert, weight);
        if (lane < a.top_k) {
            const uint64_t p = (uint64_t)(token0 + t) * a.top_k + lane;
            // What the last one reads is stored and loaded at the scope of the device, which passes by the L2 of an XCD; once the stores are done (vmcnt(0), then the
            // barrier), the counter needs no order of its own.  With one, each work-group wrote back and dropped its XCD's L2: moe_down_kernel 10.8 us for 7.4 (1 token,
            // 8 of 64 experts of 2048 x 1024, 4 bits).
            __hip_atomic_store(a.chosen + p, expert, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(a.chosen_weights + p, weight, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (a.ids) a.ids[p] = (int)expert;
            if (a.weights) a.weights[p] = weight;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const uint32_t groups = (tokens + kSelectTokens - 1) / kSelectTokens;
    if (threadIdx.x == 0) last = blockIdx.x < groups && __hip_atomic_fetch_add(a.selected + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == groups;
    __syncthreads();
    if (!last) return;
    const Selection sel = selection_at(lds, most_pairs, a.experts);
    for (uint32_t p = threadIdx.x; p < pairs; p += blockDim.x) {
        sel.id[p] = (uint16_t)__hip_atomic_load(a.chosen + (uint64_t)token0 * a.top_k + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sel.weight[p] = __hip_atomic_load(a.chosen_weights + (uint64_t)token0 * a.top_k + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    make_table(a, pairs, sel, table_at(table_of_row(a, row), most_pairs, a.most_jobs));
}

// A row's table, in LDS.
__device__ inline Table stage_table(const MoeArgs &a, uint32_t row, char *lds)
{
    const uint32_t most_pairs = min(kTokens, a.tokens) * a.top_k, bytes = table_bytes(most_pairs, a.most_jobs);
    const char *const from = table_of_row(a, row);
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<u32x4 *>(lds + i) = *reinterpret_cast<const u32x4 *>(from + i);
    __syncthreads();
    return table_at(lds, most_pairs, a.most_jobs);
}

// Tokens that every work-group of the first product selects for itself, a wavefront each: a launch less (8 tokens, 8 of 64 experts of 2048 x 1024 in 4 bits: 59.9 us, with
// a launch for it 61.4).
constexpr uint32_t kSelfSelect = 8;
constexpr int kMoeWaves = 8;                    // or as many as fit the LDS

// The scales of an expert's row for the lanes of a job.
template <typename T, bool W4, bool ZEROS, typename Job>
__device__ inline void scale_row(Job &j, int f, const MoeMatrix &m, uint32_t expert, uint64_t row)
{
    if constexpr (W4) {
        j.scales[f] = static_cast<const T *>(m.w4.scales) + (int64_t)expert * m.stride_scales + row * m.w4.lds;
        if constexpr (ZEROS) j.zeros[f] = m.w4.zeros + (int64_t)expert * m.stride_zeros + row * m.w4.ldz;
    }
}

// A unit of work: h of one job, 16 of its elements: 16 rows of gate and the same of up, `hidden` shared by the wavefronts.  A work-group takes a run of units, one
// behind the other without a pause in its loads: the wavefronts meet once a unit, over two sets of sums in turn.
// Bound by the weights' stream, and before that by the selection where it makes that itself (8 us): 8 tokens of 2048 x 1024 in 4 bits, 42 of 64 experts' 88 MB, 36 us
// with the selection of 8; 1 token in bf16, 67 MB, 20 us.  Requests of scales, a line a row, are two fifths of all.
template <typename T, bool W4, int N2, int FOLD, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(kMoeWaves * 64) moe_gate_up_kernel(const MoeArgs a)
{
    using namespace stream;
    typedef Stream<T, W4, N2, 2, 1, FOLD, ZEROS, DEPTH> S;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t tiles = (a.inner + 15) / 16, token0 = blockIdx.y * kTokens;
    float *const sums = reinterpret_cast<float *>(lds + waves * S::LDS_BYTES);           // [set][wavefront][tile][..]
    char *const table_lds = reinterpret_cast<char *>(sums + 2 * waves * S::SET_FLOATS);
    Table table;
    if (a.tokens <= kSelfSelect) {
        // A few tokens are selected by every work-group for itself, in less than another launch takes; one of them leaves the table to the next kernel.
        const uint32_t most_pairs = a.tokens * a.top_k;
        table = table_at(table_lds, most_pairs, a.most_jobs);
        const Selection sel = selection_at(lds, most_pairs, a.experts);                 // (where the rings will be)
        for (uint32_t t = wave; t < a.tokens; t += waves) {
            uint32_t expert;
            float weight;
            select_token(a, t, lane, expert, weight);
            if ((uint32_t)lane < a.top_k) {
                const uint32_t p = t * a.top_k + lane;
                sel.id[p] = (uint16_t)expert;
                sel.weight[p] = weight;
                if (blockIdx.x == 0 && a.ids) a.ids[p] = (int)expert;
                if (blockIdx.x == 0 && a.weights) a.weights[p] = weight;
            }
        }
        make_table(a, most_pairs, sel, table);
        __syncthreads();
        if (blockIdx.x == 0) {
            const uint32_t bytes = table_bytes(most_pairs, a.most_jobs);
            for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<u32x4 *>(a.table + i) = *reinterpret_cast<const u32x4 *>(table_lds + i);
        }
    } else {
        table = stage_table(a, blockIdx.y, table_lds);
    }
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < a.down_tiles; i += gridDim.x * blockDim.x) a.arrived[blockIdx.y * a.down_tiles + i] = 0;
    const uint32_t units = *table.count * tiles;
    const uint32_t unit0 = (uint32_t)((uint64_t)units * blockIdx.x / gridDim.x), unit1 = (uint32_t)((uint64_t)units * (blockIdx.x + 1) / gridDim.x);
    auto enter = [&](uint32_t u, typename S::Job &j) {
        const uint32_t job = (unit0 + u) / tiles, row0 = (unit0 + u) % tiles * 16;
        const uint32_t expert = table.expert[job], first = table.first[job], columns = table.first[job + 1] - first;
#pragma unroll
        for (int f = 0; f < 2; ++f) {            // gate, up
            const uint64_t part = (uint64_t)f * a.inner;
#pragma unroll
            for (int q = 0; q < S::WP; ++q)
                j.w[f][q] = a.gate_up.w4.q + (int64_t)expert * a.gate_up.stride + (part + min(row0 + S::load_row(lane, q), a.inner - 1)) * a.gate_up.w4.ldq;
            scale_row<T, W4, ZEROS>(j, f, a.gate_up, expert, part + min(row0 + (lane & 15), a.inner - 1));
        }
#pragma unroll
        for (int q = 0; q < S::XP; ++q) {
            const uint32_t col = S::load_column(lane, q);
            j.x_here[q] = col < columns;
            j.x[0][q] = static_cast<const T *>(a.x) + (token0 + table.pair[first + min(col, columns - 1)] / a.top_k) * a.ldx;
        }
    };
    auto flush = [&](uint32_t u, const typename S::Sums &acc) {
        float *const set = sums + (u & 1) * waves * S::SET_FLOATS;
        S::put(set + wave * S::SET_FLOATS, acc, lane);
        S::meet();
        const uint32_t job = (unit0 + u) / tiles, row0 = (unit0 + u) % tiles * 16, first = table.first[job], columns = table.first[job + 1] - first;
        for (uint32_t at = threadIdx.x; at < N2 * 16; at += blockDim.x) {
            const uint32_t i = row0 + (at & 15), col = at >> 4;
            if (i >= (kWhole<W4, N2> ? (a.inner + 7) / 8 * 8 : a.inner) || col >= columns) continue;
            const float g = S::total(set, 0, at & 15, col, waves), up = S::total(set, 1, at & 15, col, waves);
            float h = g / (1.0f + expf(-g)) * up;
            bf16_t *to = a.h + ((uint64_t)token0 * a.top_k + table.pair[first + col]) * a.ld_h;
            const uint64_t plane = (uint64_t)a.tokens * a.top_k * a.ld_h;
            if constexpr (kWhole<W4, N2>) {
                reinterpret_cast<float *>(to + (i / 4 & 1) * plane + i / 8 * 8)[i % 4] = i < a.inner ? h : 0.0f;        // (whole eights are loaded)
            } else {
                to += i;
#pragma unroll
                for (int p = 0; p < kPlanes; ++p, to += plane) {
                    const float part = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, h) & 0xFFFF0000u);     // (cut off, not rounded: no infinity comes of it)
                    *to = (bf16_t)part;
                    h = __builtin_isfinite(h) ? h - part : 0.0f;
                }
            }
        }
    };
    const uint32_t blocks = S::blocks_of(a.hidden), each = blocks / waves, more = blocks % waves, mine = each + (wave < more);
    S s(a.hidden, a.group / kW4Group, wave * each + min(wave, more), mine, lds + wave * S::LDS_BYTES, lane);
    if (mine != 0) {
        s.run(0, (unit1 - unit0) * mine, enter, flush);
    } else {                                                                            // more wavefronts than blocks: nothing to add
        typename S::Sums none;
        S::clear(none);
        for (uint32_t u = 0; u < unit1 - unit0; ++u) flush(u, none);
    }
}

// The stream of the second product.  Planes of up to four columns stand beside them as columns of their own, which the MFMAs have room for: plane p of column c is column
// c + p * N2.  Sixteen columns' planes go into one sum, and 4-bit weights into it as exact code - zero: zero points that come off later would take bits from the smaller planes
// (beside each other each plane has a sum of its own: 8 tokens of 2048 x 1024 59.8 us with exact numbers, 58.6 without).
template <typename T, bool W4, int N2, int FT, int FOLD, bool ZEROS, int DEPTH>
struct DownStream {
    static constexpr bool SIDE = N2 <= 4;
    static constexpr int PLANES = SIDE ? 1 : kWhole<W4, N2> ? 2 : kPlanes;
    typedef stream::Stream<T, W4, SIDE ? 4 * N2 : N2, FT, PLANES, FOLD, ZEROS, DEPTH, bf16_t, !SIDE, kWhole<W4, N2>> S;
};

// A work-group: 16 * FT elements of y of its tokens: the same rows of down of every expert that was selected, the jobs' blocks one behind the other and shared
// by the wavefronts.  What a wavefront has of a job goes to its own sums of all tokens; those are added in the order of the wavefronts.
// Where that is too few work-groups for the chip, several (the grid's z) share the blocks: each leaves its sums in memory, and the one that is done last adds
// them up, in the order of their numbers.  The counters that tell it were cleared by the kernel before.
// Bound by the weights' stream and, in 4 bits, by h beside it (4 columns in three planes are 3 KB to a KB of weights): 8 tokens of 2048 x 1024, 44 MB in 21 us; 1 token in
// bf16, 34 MB in 9.5 us; 64 tokens of 4096 x 2048, 268 MB in 61 us, in 4 bits 69 MB in 46.  Twice as many work-groups to a tile: 24.0 for 20.7 and 10.7 for 10.2 (h in two planes then).
template <typename T, bool W4, int N2, int FT, int FOLD, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(kMoeWaves * 64) moe_down_kernel(const MoeArgs a)
{
    using namespace stream;
    typedef DownStream<T, W4, N2, FT, FOLD, ZEROS, DEPTH> Down;
    typedef typename Down::S S;
    constexpr bool SIDE = Down::SIDE;
    constexpr int NT = S::NT, ROWS = 16 * FT;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t row0 = blockIdx.x * ROWS, token0 = blockIdx.y * kTokens, tokens = min(kTokens, a.tokens - token0), most_tokens = min(kTokens, a.tokens);
    float *const all = reinterpret_cast<float *>(lds + waves * S::LDS_BYTES);            // [wavefront][token][row]
    const Table table = stage_table(a, blockIdx.y, reinterpret_cast<char *>(all + waves * most_tokens * ROWS));
    float *const mine = all + wave * most_tokens * ROWS;
    for (uint32_t i = lane; i < most_tokens * ROWS; i += 64) mine[i] = 0.0f;
    auto enter = [&](uint32_t job, typename S::Job &j) {
        const uint32_t expert = table.expert[job], first = table.first[job], columns = table.first[job + 1] - first;
#pragma unroll
        for (int f = 0; f < FT; ++f) {
#pragma unroll
            for (int q = 0; q < S::WP; ++q)
                j.w[f][q] = a.down.w4.q + (int64_t)expert * a.down.stride + (uint64_t)min(row0 + f * 16 + S::load_row(lane, q), a.hidden - 1) * a.down.w4.ldq;
            scale_row<T, W4, ZEROS>(j, f, a.down, expert, min(row0 + f * 16 + (lane & 15), a.hidden - 1));
        }
#pragma unroll
        for (int q = 0; q < S::XP; ++q) {
            const uint32_t loaded = S::load_column(lane, q), col = SIDE ? loaded % N2 : loaded, plane = SIDE ? loaded / N2 : 0;
            j.x_here[q] = col < columns && plane < kPlanes;
            const uint64_t planes = (uint64_t)a.tokens * a.top_k * a.ld_h;
            const bf16_t *h = a.h + ((uint64_t)token0 * a.top_k + table.pair[first + min(col, columns - 1)]) * a.ld_h + min(plane, (uint32_t)kPlanes - 1) * planes;
#pragma unroll
            for (int p = 0; p < Down::PLANES; ++p) j.x[p][q] = h + p * planes;
        }
    };
    auto flush = [&](uint32_t job, const typename S::Sums &acc) {
        const uint32_t first = table.first[job], columns = table.first[job + 1] - first;
        auto add = [&](uint32_t col, int f, float v) { mine[table.pair[first + col] / a.top_k * ROWS + f * 16 + (lane & 15)] += table.weight[first + col] * v; };
        if constexpr (SIDE) {                    // the planes' sums, smallest first: of one column those of a lane, of four the same lane's of each row of 16
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int r = 0; r < N2; ++r) {
                    const float v = N2 == 1 ? acc[0][f][2] + acc[0][f][1] + acc[0][f][0]
                                            : __shfl(acc[0][f][r], lane % 16 + 32) + __shfl(acc[0][f][r], lane % 16 + 16) + acc[0][f][r];
                    if (lane < 16 && (uint32_t)r < columns) add(r, f, v);
                }
        } else {
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t col = c * 16 + (lane >> 4) * 4 + r;
                    if (col < columns)
#pragma unroll
                        for (int f = 0; f < FT; ++f) add(col, f, acc[c][f][r]);
                }
        }
    };
    const uint32_t per_job = S::blocks_of(a.inner);
    S s(a.inner, a.group / kW4Group, 0, per_job, lds + wave * S::LDS_BYTES, lane);
    const uint32_t blocks = per_job * *table.count, sharers = waves * gridDim.z, sharer = blockIdx.z * waves + wave, each = blocks / sharers, more = blocks % sharers;
    s.run(sharer * each + min(sharer, more), each + (sharer < more), enter, flush);
    __syncthreads();
    const uint32_t sums = tokens * ROWS, tile = blockIdx.y * gridDim.x + blockIdx.x;
    float *const parts = a.parts + (uint64_t)tile * gridDim.z * most_tokens * ROWS;
    if (gridDim.z > 1) {
        for (uint32_t at = threadIdx.x; at < sums; at += blockDim.x) {
            float v = 0.0f;
            for (uint32_t w = 0; w < waves; ++w) v += all[w * most_tokens * ROWS + at];
            // (as the selection's)
            __hip_atomic_store(parts + blockIdx.z * most_tokens * ROWS + at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t *const last = reinterpret_cast<uint32_t *>(lds);
        if (threadIdx.x == 0) *last = __hip_atomic_fetch_add(a.arrived + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == gridDim.z;
        __syncthreads();
        if (!*last) return;
    }
    for (uint32_t at = threadIdx.x; at < sums; at += blockDim.x) {
        const uint32_t i = row0 + at % ROWS, t = at / ROWS;
        if (i >= a.hidden) continue;
        float v = 0.0f;
        if (gridDim.z > 1)
            for (uint32_t z = 0; z < gridDim.z; ++z) v += __hip_atomic_load(parts + z * most_tokens * ROWS + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else
            for (uint32_t w = 0; w < waves; ++w) v += all[w * most_tokens * ROWS + at];
        v *= a.alpha;
        T *y = static_cast<T *>(a.y) + (token0 + t) * a.ldy + i;
        if (a.beta != 0.0f) v = __builtin_fmaf(a.beta, (float)*y, v);
        *y = (T)v;
    }
}

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
    if (l->hidden == 0 || l->hidden > MMBO_MOE_MAX_DIM || l->inner == 0 || l->inner > MMBO_MOE_MAX_DIM) return MMBO_ERR_INVALID_SIZE;
    if (l->experts == 0 || l->experts > MMBO_MOE_MAX_EXPERTS || l->top_k == 0 || l->top_k > MMBO_MOE_MAX_TOP_K || l->top_k > l->experts)
        return MMBO_ERR_INVALID_SIZE;
    if (l->group % kW4Group != 0 || l->group > kMaxDim || l->ld_router > kMaxDim || l->ld_router < l->hidden) return MMBO_ERR_INVALID_SIZE;
    if (int rc = check_matrix(l->gate_up, l->hidden, l->group)) return rc;
    return check_matrix(l->down, l->inner, l->group);
}

// (whole memory lines: rows of h that share lines with others cost the last product 74 us instead of 60, 64 tokens of 16 x 4096 x 2048)
size_t lines(size_t n) { return (n + 127) / 128 * 128; }

// Columns side by side in a stream for so many tokens, and the most jobs that a row of them can make: every job but an expert's last is full.
// Sixteen take their places in LDS and their loads whether they are there or not; with two pairs to an expert on average one in twenty experts has more than four and
// is read twice.  (8 tokens, 8 of 64 experts of 2048 x 1024 in 4 bits: 64 us in fours, 71 in sixteens)
uint32_t columns_of(const mmbo_moe_layer &l, size_t tokens)
{
    if (tokens == 1) return 1;
    return tokens <= 4 || std::min<size_t>(tokens, kTokens) * l.top_k <= 2 * l.experts ? 4 : 16;
}
uint32_t most_jobs_of(const mmbo_moe_layer &l, size_t tokens)
{
    const uint32_t pairs = std::min<uint32_t>((uint32_t)tokens, kTokens) * (uint32_t)l.top_k;
    return std::min<uint32_t>(pairs, (uint32_t)l.experts + pairs / columns_of(l, tokens));
}

// Rows of y to a tile, / 16.  16 columns of h in three planes are 12 KB to a KB of 4-bit weights, in tiles of 32 rows 6: 64 tokens, 2 of 16 experts of 4096 x 2048 101 us, in tiles
// of 16 rows 108; 32 tokens, 8 of 64 of 2048 x 1024 107 and 118; 20 tokens, 4 of 12 of 1000 x 2000 61 and 58.
constexpr int down_ft(bool w4, uint32_t columns) { return w4 && columns == 16 ? 2 : 1; }
size_t down_rows(const mmbo_moe_layer &l, size_t tokens) { return 16 * down_ft(l.group != 0, columns_of(l, tokens)); }
// Work-groups that share a tile of y: as many as make one for each of 256 CUs, up to eight.
uint32_t sharers_of(const mmbo_moe_layer &l, size_t tokens)
{
    const size_t tiles = ceil_div(l.hidden, down_rows(l, tokens)) * ceil_div(tokens, kTokens);
    return (uint32_t)std::min<size_t>(std::max<size_t>(256 / tiles, 1), 8);
}

// Places of the workspace's parts, in bytes.
struct Parts {
    size_t logits, table, chosen, chosen_weights, selected, arrived, parts, h, all, ld_h;
};
Parts parts_of(const mmbo_moe_layer &l, size_t tokens)
{
    Parts p;
    p.ld_h = (l.inner + 63) / 64 * 64;
    p.logits = 0;
    p.table = p.logits + lines(tokens * l.experts * sizeof(double));
    p.chosen = p.table + lines(ceil_div(tokens, kTokens) * table_bytes((uint32_t)(std::min<size_t>(tokens, kTokens) * l.top_k), most_jobs_of(l, tokens)));
    const size_t rows = down_rows(l, tokens), tiles = ceil_div(l.hidden, rows) * ceil_div(tokens, kTokens);
    p.chosen_weights = p.chosen + lines(tokens * l.top_k * sizeof(uint32_t));
    p.selected = p.chosen_weights + lines(tokens * l.top_k * sizeof(float));
    p.arrived = p.selected + lines(ceil_div(tokens, kTokens) * sizeof(uint32_t));
    p.parts = p.arrived + lines(tiles * sizeof(uint32_t));
    const uint32_t sharers = sharers_of(l, std::max<size_t>(tokens, 1));
    p.h = p.parts + lines(sharers > 1 ? tiles * sharers * std::min<size_t>(tokens, kTokens) * rows * sizeof(float) : 0);
    p.all = p.h + lines(kPlanes * tokens * l.top_k * p.ld_h * sizeof(bf16_t));
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

template <typename T, bool W4, int N2, int FOLD, bool ZEROS>
hipError_t launch_gate_up(const MoeArgs &a, hipStream_t s)
{
    constexpr int DEPTH = N2 < 16 && !W4 ? 3 : 2;
    typedef stream::Stream<T, W4, N2, 2, 1, FOLD, ZEROS, DEPTH> S;
    static std::atomic<bool> set[64];
    auto kernel = moe_gate_up_kernel<T, W4, N2, FOLD, ZEROS, DEPTH>;
    if (hipError_t e = allow_lds(kernel, set)) return e;
    const unsigned table = table_bytes(std::min(a.tokens, kTokens) * a.top_k, a.most_jobs), wave = S::LDS_BYTES + 2 * S::SET_FLOATS * 4;
    const unsigned waves = std::min<unsigned>(kMoeWaves, (kLds - table) / wave), bytes = waves * wave + table, held = 256 * std::min<unsigned>(kLds / bytes, 2);
    const unsigned groups = (unsigned)std::min<size_t>(a.most_jobs * ceil_div(a.inner, 16), held);
    return launch_args(kernel, dim3(groups, (unsigned)ceil_div(a.tokens, kTokens)), dim3(waves * 64), bytes, s, a);
}

template <typename T, bool W4, int N2, int FOLD, bool ZEROS>
hipError_t launch_down(const MoeArgs &a, hipStream_t s)
{
    constexpr int DEPTH = N2 == 1 ? 5 : N2 == 4 ? W4 ? 3 : 4 : 2, FT = down_ft(W4, N2);
    typedef typename DownStream<T, W4, N2, FT, FOLD, ZEROS, DEPTH>::S S;
    static std::atomic<bool> set[64];
    auto kernel = moe_down_kernel<T, W4, N2, FT, FOLD, ZEROS, DEPTH>;
    if (hipError_t e = allow_lds(kernel, set)) return e;
    const uint32_t most_tokens = std::min(a.tokens, kTokens);
    const unsigned table = table_bytes(most_tokens * a.top_k, a.most_jobs), wave = S::LDS_BYTES + most_tokens * 16 * FT * 4;
    const unsigned waves = std::min<unsigned>(kMoeWaves, (kLds - table) / wave);
    return launch_args(kernel, dim3(a.down_tiles, (unsigned)ceil_div(a.tokens, kTokens), a.sharers), dim3(waves * 64), waves * wave + table, s, a);
}

template <typename T, bool W4, int N2, int FOLD>
hipError_t launch_experts(const MoeArgs &a, hipStream_t s)
{
    hipError_t e = hipSuccess;
    if constexpr (W4) {
        e = a.gate_up.w4.zeros ? launch_gate_up<T, W4, N2, FOLD, true>(a, s) : launch_gate_up<T, W4, N2, FOLD, false>(a, s);
        if (e != hipSuccess) return e;
        return a.down.w4.zeros ? launch_down<T, W4, N2, FOLD, true>(a, s) : launch_down<T, W4, N2, FOLD, false>(a, s);
    } else {
        e = launch_gate_up<T, W4, N2, FOLD, false>(a, s);
        return e != hipSuccess ? e : launch_down<T, W4, N2, FOLD, false>(a, s);
    }
}

template <typename T, int N2>
hipError_t launch_columns(const MoeArgs &a, hipStream_t s)
{
    if (!a.group) return launch_experts<T, false, N2, 128>(a, s);
    if (a.group % 128 == 0) return launch_experts<T, true, N2, 128>(a, s);
    if (a.group % 64 == 0) return launch_experts<T, true, N2, 64>(a, s);
    return launch_experts<T, true, N2, 32>(a, s);
}

template <typename T>
hipError_t run(const MoeArgs &a, bool router32, hipStream_t s)
{
    const dim3 logits(a.experts, (unsigned)ceil_div(a.tokens, kLogitTokens));
    hipError_t e = router32 ? launch_args(moe_logits_kernel<T, float>, logits, dim3(256), 0, s, a)
                            : launch_args(moe_logits_kernel<T, T>, logits, dim3(256), 0, s, a);
    if (e != hipSuccess) return e;
    if (a.tokens > kSelfSelect) {
        const uint32_t most_tokens = std::min(a.tokens, kTokens);
        e = launch_args(moe_select_kernel, dim3((unsigned)ceil_div(most_tokens, kSelectTokens), (unsigned)ceil_div(a.tokens, kTokens)), dim3(kSelectTokens * 64),
                        select_bytes(most_tokens * a.top_k, a.experts), s, a);
        if (e != hipSuccess) return e;
    }
    return a.columns == 1 ? launch_columns<T, 1>(a, s) : a.columns == 4 ? launch_columns<T, 4>(a, s) : launch_columns<T, 16>(a, s);
}

}  // namespace
}  // namespace mmbo

using namespace mmbo;

extern "C" {

size_t mmbo_moe_workspace_bytes(const mmbo_moe_layer *layer, size_t tokens)
{
    if (check_layer(layer) != MMBO_OK || tokens > MMBO_MOE_MAX_TOKENS) return 0;
    size_t most = 16;                           // (fewer tokens may need more: they are laid out in other tiles and jobs)
    for (size_t t = 1; t <= tokens; ++t) most = std::max(most, parts_of(*layer, t).all);
    return most;
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
    a.h = reinterpret_cast<bf16_t *>(ws + p.h);
    a.ld_h = (uint32_t)p.ld_h;
    a.table = ws + p.table;
    a.chosen = reinterpret_cast<uint32_t *>(ws + p.chosen);
    a.chosen_weights = reinterpret_cast<float *>(ws + p.chosen_weights);
    a.selected = reinterpret_cast<uint32_t *>(ws + p.selected);
    a.arrived = reinterpret_cast<uint32_t *>(ws + p.arrived);
    a.parts = reinterpret_cast<float *>(ws + p.parts);
    a.down_tiles = (uint32_t)ceil_div(l.hidden, down_rows(l, tokens));
    a.sharers = sharers_of(l, tokens);
    a.ids = ids;
    a.weights = weights;
    a.columns = columns_of(l, tokens);
    a.most_jobs = most_jobs_of(l, tokens);
    a.tokens = (uint32_t)tokens; a.hidden = (uint32_t)l.hidden; a.inner = (uint32_t)l.inner; a.experts = (uint32_t)l.experts;
    a.top_k = (uint32_t)l.top_k; a.group = (uint32_t)l.group;
    a.sigmoid = l.scoring == MMBO_MOE_SIGMOID; a.renormalize = l.renormalize != 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool router32 = l.router_dtype == MMBO_F32;
    const hipError_t e = l.dtype == MMBO_F16 ? run<half_t>(a, router32, s) : run<bf16_t>(a, router32, s);
    return e == hipSuccess ? MMBO_OK : report_hip_error(e);
}

}  // extern "C"
