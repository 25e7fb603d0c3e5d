// C ABI of the mixture-of-experts layer for a few tokens: argument checks, workspace, launches and kernels.
#include "../../include/mmbo_gemm.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "stream.hpp"

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
    void *h;                                    // [2][tokens * top_k][ld_h], of the layer's type
    char *table;                                // of each row of tokens
    int *ids;                                   // [tokens][top_k]; either may be null
    float *weights;
    float alpha, beta;
    uint32_t tokens, hidden, inner, experts, top_k, group;
    uint32_t ld_h, columns, most_jobs;
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
constexpr uint32_t kLogitTokens = 4;
template <typename T, typename TR>
__global__ void __launch_bounds__(256) moe_logits_kernel(const MoeArgs a)
{
    __shared__ double parts[4][kLogitTokens];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x, t0 = blockIdx.y * kLogitTokens;
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

// Up to kTokens tokens are worked on at a time (a row of the grids).  Their (token, slot) pairs by expert, and each expert's pairs in jobs of up to `columns`.
constexpr uint32_t kTokens = 64;
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

// A work-group: the selection of a row's tokens, a wavefront a token at a time, and the row's table.  PER: experts a lane has, lane + 64 * b.
template <int PER>
__global__ void __launch_bounds__(1024) moe_select_kernel(const MoeArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t token0 = blockIdx.x * kTokens, tokens = min(kTokens, a.tokens - token0), pairs = tokens * a.top_k, most_pairs = min(kTokens, a.tokens) * a.top_k;
    float *const weight = reinterpret_cast<float *>(lds);                               // by token and slot
    uint16_t *const id = reinterpret_cast<uint16_t *>(weight + most_pairs), *const before = id + most_pairs, *const jobs_before = before + a.experts;
    for (uint32_t t = wave; t < tokens; t += waves) {
        const double *logits = a.logits + (uint64_t)(token0 + t) * a.experts;
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
        double sum = 0.0, highest = 0.0;
        if (!a.sigmoid) {
            // (a NaN among the logits is no largest one; it makes the sum NaN, which scores that only count against each other do not need)
            most = wave_max(most);
            highest = __builtin_bit_cast(double, most >> 63 ? most & ~(1ull << 63) : ~most);
            if (!a.renormalize || a.bias) {
#pragma unroll
                for (int b = 0; b < PER; ++b)
                    if (lane + 64 * b < a.experts) sum += exp(logit[b] - highest);
                sum = wave_sum(sum);
            }
        }
        // (not over its sum where only selected scores count against each other)
        auto score = [&](double v) { return a.sigmoid ? 1.0 / (1.0 + exp(-v)) : !a.renormalize || a.bias ? exp(v - highest) / sum : exp(v - highest); };
        if (a.bias)
#pragma unroll
            for (int b = 0; b < PER; ++b)
                if (lane + 64 * b < a.experts) key[b] = order_of(score(logit[b]) + (double)a.bias[lane + 64 * b]);
        uint32_t mine = 0, here = 0;             // the expert of slot `lane`; of this lane's experts, those that may still be taken
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
            bool found = false;
#pragma unroll
            for (int b = 0; b < PER; ++b) {
                const uint64_t who = __ballot((here >> b & 1) && key[b] == best);
                if (!found && who != 0) {
                    e = 64 * b + __builtin_ctzll(who);
                    found = true;
                }
            }
            if (lane == (e & 63)) here &= ~(1u << (e >> 6));
            if (lane == s) mine = e;
        }
        double v = lane < a.top_k ? score(logits[mine]) : 0.0;
        if (a.renormalize) {
            const double total = wave_sum(v);
            v = total == 0.0 ? 0.0 : v / total;
        }
        if (lane < a.top_k) {
            const uint32_t p = t * a.top_k + lane;
            id[p] = (uint16_t)mine;
            weight[p] = (float)v;
            if (a.ids) a.ids[(uint64_t)token0 * a.top_k + p] = (int)mine;
            if (a.weights) a.weights[(uint64_t)token0 * a.top_k + p] = (float)v;
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.experts; e += blockDim.x) {
        uint32_t n = 0;
        for (uint32_t p = 0; p < pairs; ++p) n += id[p] == e;
        before[e] = (uint16_t)n;
        jobs_before[e] = (uint16_t)((n + a.columns - 1) / a.columns);
    }
    __syncthreads();
    const Table table = table_at(a.table + (uint64_t)blockIdx.x * table_bytes(most_pairs, a.most_jobs), most_pairs, a.most_jobs);
    if (threadIdx.x < 64) {                      // sums of those in front
        uint32_t n0 = 0, j0 = 0;
        for (uint32_t e0 = 0; e0 < a.experts; e0 += 64) {
            const uint32_t e = e0 + threadIdx.x;
            const uint32_t n = e < a.experts ? before[e] : 0, j = e < a.experts ? jobs_before[e] : 0;
            uint32_t ns = n, js = j;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t nn = __shfl_up(ns, d), jj = __shfl_up(js, d);
                if ((int)threadIdx.x >= d) { ns += nn; js += jj; }
            }
            if (e < a.experts) {
                before[e] = (uint16_t)(n0 + ns - n);
                jobs_before[e] = (uint16_t)(j0 + js - j);
            }
            n0 += __shfl(ns, 63);
            j0 += __shfl(js, 63);
        }
        if (threadIdx.x == 0) {
            *table.count = j0;
            table.first[j0] = (uint16_t)pairs;
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const uint32_t from = before[e], to = e + 1 < a.experts ? before[e + 1] : pairs;
        if (from == to) continue;
        uint32_t at = from, job = jobs_before[e];
        for (uint32_t n = from; n < to; n += a.columns, ++job) {
            table.expert[job] = (uint16_t)e;
            table.first[job] = (uint16_t)n;
        }
        for (uint32_t p = 0; p < pairs; ++p)
            if (id[p] == e) {
                table.pair[at] = (uint16_t)p;
                table.weight[at++] = weight[p];
            }
    }
}

// A row's table, in LDS.
__device__ inline Table stage_table(const MoeArgs &a, uint32_t row, char *lds)
{
    const uint32_t most_pairs = min(kTokens, a.tokens) * a.top_k, bytes = table_bytes(most_pairs, a.most_jobs);
    const char *const from = a.table + (uint64_t)row * bytes;
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16) *reinterpret_cast<u32x4 *>(lds + i) = *reinterpret_cast<const u32x4 *>(from + i);
    __syncthreads();
    return table_at(lds, most_pairs, a.most_jobs);
}

constexpr int kMoeWaves = 8;                    // or as many as fit the LDS
constexpr unsigned kLds = 160 * 1024;

// A row of an expert's weight for the lanes of a job.
template <typename T, bool W4, bool ZEROS, typename Job>
__device__ inline void weight_row(Job &j, int f, const MoeMatrix &m, uint32_t expert, uint64_t load_row, uint64_t row)
{
    j.w[f] = m.w4.q + (int64_t)expert * m.stride + load_row * m.w4.ldq;
    if constexpr (W4) {
        j.scales[f] = static_cast<const T *>(m.w4.scales) + (int64_t)expert * m.stride_scales + row * m.w4.lds;
        if constexpr (ZEROS) j.zeros[f] = m.w4.zeros + (int64_t)expert * m.stride_zeros + row * m.w4.ldz;
    }
}

// Of a unit's 16 x 16 sums the columns that N2 leaves: floats of a tile, and where lane l's four lie.
template <int N2> constexpr int kTileFloats = N2 < 16 ? 16 * N2 : 256;

// A unit of work: h of one job, 16 of its elements: 16 rows of gate and the same of up, `hidden` shared by the wavefronts.  A work-group takes a run of units, one
// behind the other without a pause in its loads: the wavefronts meet once a unit, over two sets of sums in turn.
template <typename T, bool W4, int N2, int FOLDS, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(kMoeWaves * 64) moe_gate_up_kernel(const MoeArgs a)
{
    using namespace stream;
    typedef Stream<T, W4, N2, 2, 1, FOLDS, ZEROS, DEPTH> S;
    constexpr int NT = S::NT, TILE = kTileFloats<N2>, SET = NT * 2 * TILE;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t tiles = (a.inner + 15) / 16, token0 = blockIdx.y * kTokens;
    float *const sums = reinterpret_cast<float *>(lds + waves * S::LDS_BYTES);           // [set][wavefront][tile][..]
    const Table table = stage_table(a, blockIdx.y, reinterpret_cast<char *>(sums + 2 * waves * SET));
    const uint32_t units = *table.count * tiles;
    const uint32_t unit0 = (uint32_t)((uint64_t)units * blockIdx.x / gridDim.x), unit1 = (uint32_t)((uint64_t)units * (blockIdx.x + 1) / gridDim.x);
    auto enter = [&](uint32_t u, typename S::Job &j) {
        const uint32_t job = (unit0 + u) / tiles, row0 = (unit0 + u) % tiles * 16;
        const uint32_t expert = table.expert[job], first = table.first[job], columns = table.first[job + 1] - first;
        const uint32_t load_row = min(row0 + (lane >> 2), a.inner - 1), row = min(row0 + (lane & 15), a.inner - 1);
        weight_row<T, W4, ZEROS>(j, 0, a.gate_up, expert, load_row, row);
        weight_row<T, W4, ZEROS>(j, 1, a.gate_up, expert, (uint64_t)a.inner + load_row, (uint64_t)a.inner + row);
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const uint32_t col = (uint32_t)(lane >> 2) % N2 % 16 + c * 16;
            j.x_here[c] = col < columns;
            j.x[0][c] = static_cast<const T *>(a.x) + (token0 + table.pair[first + min(col, columns - 1)] / a.top_k) * a.ldx;
        }
    };
    auto flush = [&](uint32_t u, const typename S::Sums &acc) {
        float *const set = sums + (u & 1) * waves * SET;
        if (N2 >= 16 || lane < 16) {
#pragma unroll
            for (int t = 0; t < NT * 2; ++t) {
                const f32x4 v = acc[t / 2][t % 2];
                float *const to = set + wave * SET + t * TILE;
                if constexpr (N2 == 1) to[lane] = v[0];
                else *reinterpret_cast<f32x4 *>(to + lane * 4) = v;
            }
        }
        // (not __syncthreads(): what is under way for the next unit stays so)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint32_t job = (unit0 + u) / tiles, row0 = (unit0 + u) % tiles * 16, first = table.first[job], columns = table.first[job + 1] - first;
        for (uint32_t at = threadIdx.x; at < N2 * 16; at += blockDim.x) {
            const uint32_t i = row0 + (at & 15), col = at >> 4;
            if (i >= a.inner || col >= columns) continue;
            const uint32_t place = N2 == 1 ? at & 15 : (col >> 4) * 2 * TILE + ((col >> 2 & 3) * 16 + (at & 15)) * 4 + (col & 3);
            float g = 0.0f, up = 0.0f;
            for (uint32_t w = 0; w < waves; ++w) {
                g += set[w * SET + place];
                up += set[w * SET + TILE + place];
            }
            const float h = g / (1.0f + expf(-g)) * up;
            T *const to = static_cast<T *>(a.h) + ((uint64_t)token0 * a.top_k + table.pair[first + col]) * a.ld_h + i;
            const T high = (T)h;
            *to = high;
            to[(uint64_t)a.tokens * a.top_k * a.ld_h] = (T)(h - (float)high);
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

// A work-group: 16 * FT elements of y of its tokens: the same rows of down of every expert that was selected, the jobs' blocks one behind the other and shared
// by the wavefronts.  What a wavefront has of a job goes to its own sums of all tokens; those are added in the order of the wavefronts.
template <typename T, bool W4, int N2, int FT, int FOLDS, bool ZEROS, int DEPTH>
__global__ void __launch_bounds__(kMoeWaves * 64) moe_down_kernel(const MoeArgs a)
{
    using namespace stream;
    typedef Stream<T, W4, N2, FT, 2, FOLDS, ZEROS, DEPTH> S;
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
        for (int f = 0; f < FT; ++f)
            weight_row<T, W4, ZEROS>(j, f, a.down, expert, min(row0 + f * 16 + (lane >> 2), a.hidden - 1), min(row0 + f * 16 + (lane & 15), a.hidden - 1));
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const uint32_t col = (uint32_t)(lane >> 2) % N2 % 16 + c * 16;
            j.x_here[c] = col < columns;
            const T *h = static_cast<const T *>(a.h) + ((uint64_t)token0 * a.top_k + table.pair[first + min(col, columns - 1)]) * a.ld_h;
            j.x[0][c] = h;
            j.x[1][c] = h + (uint64_t)a.tokens * a.top_k * a.ld_h;
        }
    };
    auto flush = [&](uint32_t job, const typename S::Sums &acc) {
        const uint32_t first = table.first[job], columns = table.first[job + 1] - first;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t col = c * 16 + (lane >> 4) * 4 + r;
                if (col < columns) {
                    const float w = table.weight[first + col];
                    float *const to = mine + table.pair[first + col] / a.top_k * ROWS + (lane & 15);
#pragma unroll
                    for (int f = 0; f < FT; ++f) to[f * 16] += w * acc[c][f][r];
                }
            }
    };
    const uint32_t per_job = S::blocks_of(a.inner);
    S s(a.inner, a.group / kW4Group, 0, per_job, lds + wave * S::LDS_BYTES, lane);
    const uint32_t blocks = per_job * *table.count, each = blocks / waves, more = blocks % waves;
    s.run(wave * each + min(wave, more), each + (wave < more), enter, flush);
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < tokens * ROWS; at += blockDim.x) {
        const uint32_t i = row0 + at % ROWS, t = at / ROWS;
        if (i >= a.hidden) continue;
        float v = 0.0f;
        for (uint32_t w = 0; w < waves; ++w) v += all[w * most_tokens * ROWS + at];
        v *= a.alpha;
        T *y = static_cast<T *>(a.y) + (token0 + t) * a.ldy + i;
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
    if (l->hidden == 0 || l->hidden > MMBO_MOE_MAX_DIM || l->inner == 0 || l->inner > MMBO_MOE_MAX_DIM) return MMBO_ERR_INVALID_SIZE;
    if (l->experts == 0 || l->experts > MMBO_MOE_MAX_EXPERTS || l->top_k == 0 || l->top_k > MMBO_MOE_MAX_TOP_K || l->top_k > l->experts)
        return MMBO_ERR_INVALID_SIZE;
    if (l->group % kW4Group != 0 || l->group > kMaxDim || l->ld_router > kMaxDim || l->ld_router < l->hidden) return MMBO_ERR_INVALID_SIZE;
    if (int rc = check_matrix(l->gate_up, l->hidden, l->group)) return rc;
    return check_matrix(l->down, l->inner, l->group);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// Columns side by side in a stream for so many tokens, and the most jobs that a row of them can make: every job but an expert's last is full.
uint32_t columns_of(uint32_t tokens) { return tokens == 1 ? 1 : tokens <= 4 ? 4 : 16; }
uint32_t most_jobs_of(const mmbo_moe_layer &l, size_t tokens)
{
    const uint32_t pairs = std::min<uint32_t>((uint32_t)tokens, kTokens) * (uint32_t)l.top_k;
    return std::min<uint32_t>(pairs, (uint32_t)l.experts + pairs / columns_of((uint32_t)tokens));
}

// Places of the workspace's parts, in bytes.
struct Parts {
    size_t logits, table, h, all, ld_h;
};
Parts parts_of(const mmbo_moe_layer &l, size_t tokens)
{
    Parts p;
    p.ld_h = (l.inner + 7) / 8 * 8;
    p.logits = 0;
    p.table = p.logits + round16(tokens * l.experts * sizeof(double));
    p.h = p.table + ceil_div(tokens, kTokens) * table_bytes((uint32_t)(std::min<size_t>(tokens, kTokens) * l.top_k), most_jobs_of(l, tokens));
    p.all = p.h + round16(2 * tokens * l.top_k * p.ld_h * sizeof(half_t));
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

template <typename T, bool W4, int N2, int FOLDS, bool ZEROS>
hipError_t launch_experts(const MoeArgs &a, hipStream_t s)
{
    constexpr int UP_DEPTH = N2 < 16 ? 3 : 2, DEPTH = N2 == 1 ? 5 : N2 == 4 ? 4 : 2, FT = 1;
    typedef stream::Stream<T, W4, N2, 2, 1, FOLDS, ZEROS, UP_DEPTH> Up;
    typedef stream::Stream<T, W4, N2, FT, 2, FOLDS, ZEROS, DEPTH> Down;
    const uint32_t rows = (uint32_t)ceil_div(a.tokens, kTokens), most_tokens = std::min(a.tokens, kTokens);
    const unsigned table = table_bytes(most_tokens * a.top_k, a.most_jobs);
    static std::atomic<bool> set[2][64];
    auto up = moe_gate_up_kernel<T, W4, N2, FOLDS, ZEROS, UP_DEPTH>;
    auto down = moe_down_kernel<T, W4, N2, FT, FOLDS, ZEROS, DEPTH>;
    if (hipError_t e = allow_lds(up, set[0])) return e;
    if (hipError_t e = allow_lds(down, set[1])) return e;
    const unsigned up_wave = Up::LDS_BYTES + 2 * Up::NT * 2 * kTileFloats<N2> * 4, down_wave = Down::LDS_BYTES + most_tokens * 16 * FT * 4;
    const unsigned up_waves = std::min<unsigned>(kMoeWaves, (kLds - table) / up_wave), down_waves = std::min<unsigned>(kMoeWaves, (kLds - table) / down_wave);
    const unsigned groups = (unsigned)std::min<size_t>(a.most_jobs * ceil_div(a.inner, 16), 256);
    hipError_t e = launch_args(up, dim3(groups, rows), dim3(up_waves * 64), up_waves * up_wave + table, s, a);
    if (e != hipSuccess) return e;
    return launch_args(down, dim3((unsigned)ceil_div(a.hidden, 16 * FT), rows), dim3(down_waves * 64), down_waves * down_wave + table, s, a);
}

template <typename T, int N2>
hipError_t launch_columns(const MoeArgs &a, hipStream_t s)
{
    if (!a.group) return launch_experts<T, false, N2, 1, false>(a, s);
    auto folds = [&](auto n) {
        return a.gate_up.w4.zeros ? launch_experts<T, true, N2, decltype(n)::value, true>(a, s) : launch_experts<T, true, N2, decltype(n)::value, false>(a, s);
    };
    if (a.group % 128 == 0) return folds(std::integral_constant<int, 1>());
    if (a.group % 64 == 0) return folds(std::integral_constant<int, 2>());
    return folds(std::integral_constant<int, 4>());
}

hipError_t launch_select(const MoeArgs &a, hipStream_t s)
{
    const uint32_t most_tokens = std::min(a.tokens, kTokens), rows = (uint32_t)ceil_div(a.tokens, kTokens);
    const unsigned waves = std::min(most_tokens, 16u), lds = most_tokens * a.top_k * 6 + a.experts * 4;
    const dim3 block(waves * 64);
    if (a.experts <= 64) return launch_args(moe_select_kernel<1>, dim3(rows), block, lds, s, a);
    if (a.experts <= 128) return launch_args(moe_select_kernel<2>, dim3(rows), block, lds, s, a);
    return launch_args(moe_select_kernel<8>, dim3(rows), block, lds, s, a);
}

template <typename T>
hipError_t run(const MoeArgs &a, bool router32, hipStream_t s)
{
    const dim3 logits(a.experts, (unsigned)ceil_div(a.tokens, kLogitTokens));
    hipError_t e = router32 ? launch_args(moe_logits_kernel<T, float>, logits, dim3(256), 0, s, a)
                            : launch_args(moe_logits_kernel<T, T>, logits, dim3(256), 0, s, a);
    if (e != hipSuccess) return e;
    e = launch_select(a, s);
    if (e != hipSuccess) return e;
    return a.columns == 1 ? launch_columns<T, 1>(a, s) : a.columns == 4 ? launch_columns<T, 4>(a, s) : launch_columns<T, 16>(a, s);
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
    a.h = ws + p.h;
    a.ld_h = (uint32_t)p.ld_h;
    a.table = ws + p.table;
    a.ids = ids;
    a.weights = weights;
    a.columns = columns_of((uint32_t)tokens);
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
