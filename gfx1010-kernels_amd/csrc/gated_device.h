// Kernels of the gated residual norm (include/rln.h, the rln_gated_* entry
// points): a block's output, normed, gated and scaled, added to the stream,
// and the norm in front of the next block.
//
// Per row of H values (rs, bs two constants; gate and the norms' weights rows of
// H values, c = bs * gate * branch_weight):
//
//   rb = 1 / sqrt(sum(branch^2) / H + branch_eps), or 1 without a branch weight
//   u  = rs * x + c * (branch * rb), rounded to x's type
//   r  = 1 / sqrt(sum(u^2) / H + eps);    normalized = u * r * weight
//
// Backward, with v = u * r, a = branch * rb and p = gy * weight:
//
//   g           = gu + r * (p - v * sum(p * v) / H)        the gradient of u
//   grad_x      = rs * g
//   q           = c * g                                     the gradient of a
//   grad_branch = rb * (q - a * sum(q * a) / H), or q without a branch weight
//   S = g * a,  T = gy * v; their sums over the rows give, by products with rows
//   that do not depend on the token, the gradients of gate, branch_weight, weight
//
// sum(q * a) would wait for sum(p * v). With g written out it is
//
//   sum(q * a) = sum(c * a * (gu + r * p)) - r * sum(p * v) / H * sum(c * a * v)
//
// so the row's three sums are taken together, and a row costs one exchange
// between its waves instead of two.
//
// Every pass is bound by memory (about 15 fp32 operations per element forward, 40
// backward, against 6-24 bytes). Rows, waves, vectors and accesses are those of the
// root-mean-square norm (rms_device.h), whose helpers these kernels use.
//
// Measured: [16384, 4096] bf16, gate and weight by sample, forward 98 us (5.5 TB/s),
// backward 150 (5.4) and 6.4 for its sums; [6001, 2880] bf16 forward 29 (4.8); [3711,
// 1001] fp32 with a token gate 17.6 and 29.4 (4.0-4.2: rows at element alignment); [8,
// 4096] bf16 3.8. A large copy reaches 5.15.
#ifndef GATED_DEVICE_H
#define GATED_DEVICE_H

#include "rms_device.h"

namespace rln {
namespace gated {

using namespace rms;

// A row of factors (gate, weight) that `rows` consecutive rows of the stream
// share: all rows, those of a sample, or one.
struct Factor {
    const void* data;  // null: one
    int64_t stride;    // between consecutive rows of factors, in elements
    int64_t rows;
    int dtype;
    int kind;          // Repeat
    uint32_t magic;    // of a 32-bit division by `rows`
    int shift;
};

enum Repeat { kShared, kToken, kSample, kWideSample };

// A block's waves as teams of `parts`. A wave finds its own by a product: a block of
// one row would wait a good part of its time for the divisions.
struct Split {
    int parts;
    int teams;
    uint32_t inverse;  // 2^16 / parts, rounded up
};

struct ForwardArgs {
    const void* x;
    const void* branch;
    const void* branch_weight;  // null without a norm of the branch
    Factor gate;
    Factor weight;
    void* updated;
    void* normalized;
    float* statistics;  // r, then rb, [rows] each; may be null
    int64_t x_stride;
    int64_t branch_stride;
    int64_t rows;
    int hidden;
    Split split;
    int row_lanes;
    int words;
    int branch_weight_dtype;
    int output_dtype;
    float residual_scale;
    float branch_scale;
    float eps;
    float branch_eps;
    float inv_hidden;
};

struct BackwardArgs {
    const void* grad_updated;     // may be null, as grad_normalized
    const void* grad_normalized;
    const void* updated;
    const void* branch;
    const void* branch_weight;
    Factor gate;
    Factor weight;
    const float* statistics;
    void* grad_x;
    void* grad_branch;
    void* grad_gate;    // of a gate with a row for each token; else null
    float* partials;    // [units][2][hidden]: sums of S and T, or null
    int64_t branch_stride;
    int64_t rows;
    int64_t group_rows;  // rows that share their factors
    int64_t units;       // runs of rows with sums of their own
    int group_units;     // of a group
    int hidden;
    Split split;
    int row_lanes;
    int words;
    int grad_dtype;      // grad_normalized's
    int branch_weight_dtype;
    float residual_scale;
    float branch_scale;
    float inv_hidden;
};

// N elements of a type known at run time, as raw words (16-bit ones in the
// first half). Loaded and widened apart, so that a row's loads are all under way
// before the first is waited for.
template <int N>
struct RawAny {
    uint32_t words[N];
};

template <Access kAccess, int N, int Policy = kCached>
__device__ __forceinline__ RawAny<N> load_any(const void* data, int dtype, int64_t first,
                                              int column, int hidden) {
    RawAny<N> out;
    if (dtype == RLN_DTYPE_F32) {
        const auto raw = load<kAccess, float, N, Policy>(static_cast<const float*>(data) + first,
                                                         column, hidden);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            out.words[i] = raw.words[i];
        }
    } else {  // both 16-bit types are loaded alike
        const auto raw = load<kAccess, half_t, N, Policy>(static_cast<const half_t*>(data) + first,
                                                          column, hidden);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            out.words[i] = i < N / 2 ? raw.words[i] : 0;
        }
    }
    return out;
}

template <Access kAccess, int N>
__device__ __forceinline__ void widen_any(const RawAny<N>& any, int dtype, int column, int hidden,
                                          float (&out)[N]) {
    if (dtype == RLN_DTYPE_F32) {
        Raw<float, N> raw;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            raw.words[i] = any.words[i];
        }
        settle<kAccess>(raw, column, hidden);
        widen<float, N>(raw, out);
    } else {
        Raw<half_t, N> raw;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            raw.words[i] = any.words[i];
        }
        settle<kAccess>(raw, column, hidden);
        if (dtype == RLN_DTYPE_F16) {
            widen<half_t, N>(raw, out);
        } else {
            Raw<bf16_t, N> other;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                other.words[i] = raw.words[i];
            }
            widen<bf16_t, N>(other, out);
        }
    }
}

// Of a tensor that may be missing; `missing` is then every element's value.
template <Access kAccess, int N, int Policy = kCached>
__device__ __forceinline__ RawAny<N> load_optional(const void* data, int dtype, int64_t first,
                                                   int column, int hidden) {
    if (data != nullptr) {
        return load_any<kAccess, N, Policy>(data, dtype, first, column, hidden);
    }
    return RawAny<N>{};
}

template <Access kAccess, int N>
__device__ __forceinline__ void widen_optional(const RawAny<N>& raw, const void* data, int dtype,
                                               int column, int hidden, float missing,
                                               float (&out)[N]) {
    if (data != nullptr) {
        widen_any<kAccess, N>(raw, dtype, column, hidden, out);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            out[e] = missing;
        }
    }
}

// The first element of the factors' row for a row of the stream.
__device__ __forceinline__ int64_t factor_row(const Factor& factor, int64_t row) {
    if (factor.kind == kShared) {
        return 0;
    }
    int64_t index = row;
    if (factor.kind == kSample) {
        const uint32_t narrow = static_cast<uint32_t>(row);
        const uint32_t high = __umulhi(narrow, factor.magic);
        index = (high + ((narrow - high) >> 1)) >> factor.shift;
    } else if (factor.kind == kWideSample) {
        index = row / factor.rows;
    }
    return index * factor.stride;
}

__device__ __forceinline__ Team team_of(const Split& split) {
    Team team;
    team.wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    team.index = static_cast<int>(static_cast<uint32_t>(team.wave) * split.inverse >> 16);
    team.part = team.wave - team.index * split.parts;
    team.teams = split.teams;
    return team;
}

// The factors from an element on.
__device__ __forceinline__ const void* row_of(const Factor& factor, int64_t first) {
    return static_cast<const char*>(factor.data) + first * (factor.dtype == RLN_DTYPE_F32 ? 4 : 2);
}

template <Access kAccess>
__device__ __forceinline__ float row_total(float value, int row_lanes) {
    return kAccess == Access::kLanes ? lanes_sum(value, row_lanes) : wave_sum(value);
}

// ----------------------------------------------------------------------------
// Forward: one row per team and turn, as rms_device.h's.

// Waves of a block: three slots are taken for rows of at most 8 (pass_shape). The
// registers are those of four waves for each SIMD either way: a few of three slots go
// to memory, and three waves without that are slower where it matters ([1820, 9216]
// bf16 44 against 37 us).
constexpr int forward_threads(int slots) {
    return (slots == 3 ? 8 : kMaxParts) * kWave;
}

template <typename X, typename B, int V, bool kPost, Access kAccess>
__global__ __launch_bounds__(forward_threads(V), 4) void forward_kernel(ForwardArgs a) {
    constexpr int N = kColumns<X>;
    __shared__ float sums[2][2][kMaxParts];
    const Team team = team_of(a.split);
    const Place place = place_of<kAccess>(a.row_lanes);
    const int block_rows = team.teams * place.rows;
    const int64_t step = static_cast<int64_t>(gridDim.x) * block_rows;
    int turn = 0;
    // The team's total of one value per wave; every team of the block makes the
    // same number of calls. Two buffers: a wave that is ahead writes the one that
    // the slower ones do not read.
    const auto team_total = [&](float value, int which) {
        if (a.split.parts > 1) {
            sums[turn][which][team.wave] = value;
            __syncthreads();
            value = 0.0f;
            for (int part = 0; part < a.split.parts; ++part) {
                value += sums[turn][which][team.index * a.split.parts + part];
            }
        }
        return value;
    };
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * block_rows; base < a.rows;
         base += step) {
        const int64_t row = base + team.index * place.rows + place.row;
        const bool live = row < a.rows;
        const int hidden = live ? a.hidden : 0;
        const int64_t first = row * a.hidden;
        const X* x = static_cast<const X*>(a.x) + row * a.x_stride;
        const B* branch = static_cast<const B*>(a.branch) + row * a.branch_stride;
        int column[V];
        Raw<X, N> raw_x[V];
        Raw<B, N> raw_branch[V];
        RawAny<N> raw_gate[V];
        RawAny<N> raw_post[V];
        RawAny<N> raw_weight[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            column[v] = ((v * a.split.parts + team.part) * kWave + place.lane) * N;
            raw_branch[v] = load<kAccess, B, N>(branch, column[v], hidden);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            raw_x[v] = load<kAccess, X, N>(x, column[v], hidden);
        }
        const int64_t gate_row = factor_row(a.gate, live ? row : 0);
        const int64_t weight_row = factor_row(a.weight, live ? row : 0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            raw_gate[v] = load_optional<kAccess, N>(a.gate.data, a.gate.dtype, gate_row, column[v],
                                                    hidden);
            if constexpr (kPost) {
                raw_post[v] = load_any<kAccess, N>(a.branch_weight, a.branch_weight_dtype, 0,
                                                   column[v], hidden);
            }
            raw_weight[v] = load_any<kAccess, N>(a.weight.data, a.weight.dtype, weight_row,
                                                 column[v], hidden);
        }
        float u[V][N];
        float branch_rstd = 1.0f;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            settle<kAccess>(raw_branch[v], column[v], hidden);
            widen<B, N>(raw_branch[v], u[v]);
            if constexpr (kPost) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    sum += u[v][e] * u[v][e];
                }
            }
        }
        if constexpr (kPost) {
            sum = team_total(row_total<kAccess>(sum, a.row_lanes), 0);
            branch_rstd = 1.0f / __builtin_sqrtf(sum * a.inv_hidden + a.branch_eps);
        }
        X* updated = static_cast<X*>(a.updated) + first;
        sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float stream[N];
            float gate[N];
            settle<kAccess>(raw_x[v], column[v], hidden);
            widen<X, N>(raw_x[v], stream);
            widen_optional<kAccess, N>(raw_gate[v], a.gate.data, a.gate.dtype, column[v], hidden,
                                       1.0f, gate);
            float post[N];
            if constexpr (kPost) {
                widen_any<kAccess, N>(raw_post[v], a.branch_weight_dtype, column[v], hidden, post);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float factor = a.branch_scale * gate[e];
                if constexpr (kPost) {
                    factor *= post[e];
                    u[v][e] *= branch_rstd;
                }
                u[v][e] = a.residual_scale * stream[e] + factor * u[v][e];
            }
            // The norm is taken of the rounded stream, which is what the
            // backward and the next layer read.
            const Raw<X, N> rounded = narrow<X, N>(u[v]);
            store<kAccess, kForwardStores, X, N>(updated, column[v], hidden, rounded);
            widen<X, N>(rounded, u[v]);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                // Past the row's end the scaled zeros are zeros: nothing is added.
                sum += u[v][e] * u[v][e];
            }
        }
        sum = team_total(row_total<kAccess>(sum, a.row_lanes), 1);
        turn ^= 1;
        const float rstd = 1.0f / __builtin_sqrtf(sum * a.inv_hidden + a.eps);
        if (a.statistics != nullptr && live && team.part == 0 && place.lane == 0) {
            a.statistics[row] = rstd;
            if constexpr (kPost) {
                a.statistics[a.rows + row] = branch_rstd;
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float weight[N];
            widen_any<kAccess, N>(raw_weight[v], a.weight.dtype, column[v], hidden, weight);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                u[v][e] = u[v][e] * rstd * weight[e];
            }
            store_as<kAccess, kForwardStores, N>(a.normalized, a.output_dtype, first, column[v],
                                                 hidden, u[v]);
        }
    }
}

// ----------------------------------------------------------------------------
// Backward: a block's teams walk the rows of a unit, a run of rows of one group;
// each lane keeps its columns' share of the sums of S and T in registers, the block
// adds its teams' shares through LDS and writes them to the unit's row of the
// partials, which sum_units_kernel adds in a fixed order: no atomics, the same bits
// on every run.

// What a lane reads of a row.
template <typename X, typename B, int V, bool kToken>
struct Row {
    Raw<X, kColumns<X>> u[V];
    Raw<B, kColumns<X>> branch[V];
    Raw<X, kColumns<X>> grad[V];
    RawAny<kColumns<X>> upstream[V];
    RawAny<kColumns<X>> gate[kToken ? V : 1];
    float rstd;
    float branch_rstd;
};

template <typename X, typename B, int V, bool kPost, bool kToken, Access kAccess>
__device__ __forceinline__ void load_row(const BackwardArgs& a, int64_t row, int64_t end,
                                         const int (&column)[V], Row<X, B, V, kToken>* out) {
    constexpr int N = kColumns<X>;
    const bool live = row < end;
    const int hidden = live ? a.hidden : 0;
    const int64_t first = row * a.hidden;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        out->u[v] = load<kAccess, X, N>(static_cast<const X*>(a.updated) + first, column[v],
                                        hidden);
        out->branch[v] = load<kAccess, B, N>(
            static_cast<const B*>(a.branch) + row * a.branch_stride, column[v], hidden);
        out->grad[v] = Raw<X, N>{};
        if (a.grad_updated != nullptr) {
            out->grad[v] = load<kAccess, X, N>(static_cast<const X*>(a.grad_updated) + first,
                                               column[v], hidden);
        }
        out->upstream[v] = load_optional<kAccess, N, kOnce>(a.grad_normalized, a.grad_dtype, first,
                                                            column[v], hidden);
        if constexpr (kToken) {
            out->gate[v] = load_any<kAccess, N, kOnce>(a.gate.data, a.gate.dtype,
                                                       row * a.gate.stride, column[v], hidden);
        }
    }
    out->rstd = live ? a.statistics[row] : 0.0f;
    out->branch_rstd = kPost && live ? a.statistics[a.rows + row] : 1.0f;
}

// sums += a * b, of a lane's own N sums in LDS.
template <int N>
__device__ __forceinline__ void add_products(float* sums, const float (&a)[N],
                                             const float (&b)[N]) {
    typedef float Four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        Four four = *reinterpret_cast<Four*>(sums + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            four[k] = __builtin_fmaf(a[i + k], b[i + k], four[k]);
        }
        *reinterpret_cast<Four*>(sums + i) = four;
    }
}

// kToken: the gate has a row for each token, read beside the others; S then holds
// it as a factor. Otherwise the factors do not depend on the row and stay in
// registers over a unit's rows.

template <typename X, typename B, int V, bool kPost, bool kToken, Access kAccess>
__global__ __launch_bounds__(kMaxParts * kWave) void backward_kernel(BackwardArgs a) {
    constexpr int N = kColumns<X>;
    // As far as the registers go.
    constexpr bool kAhead = kAccess != Access::kLanes && V * N <= (kToken ? 4 : 8);
    // Lanes of more than 8 columns, of which a block is one row, keep the sums in LDS,
    // each its own, since they do not fit the registers.
    constexpr bool kLdsSums = V * N > 8;
    // [teams - 1][hidden], one sum at a time; or the sums [2][block's columns].
    extern __shared__ __attribute__((aligned(16))) float shares[];
    __shared__ float sums[2][3][kMaxParts];
    const Team team = team_of(a.split);
    const Place place = place_of<kAccess>(a.row_lanes);
    const int block_rows = team.teams * place.rows;
    int column[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        column[v] = ((v * a.split.parts + team.part) * kWave + place.lane) * N;
    }
    int turn = 0;
    // Every team of the block makes the same number of turns (barriers inside).
    for (int64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const int64_t group = unit / a.group_units;
        const int64_t begin = group * a.group_rows;
        const int64_t end = begin + a.group_rows;
        // The next row's loads are under way while a row is reduced and written.
        const int64_t step = static_cast<int64_t>(a.group_units) * block_rows;
        int64_t base = begin + (unit - group * a.group_units) * block_rows;
        Row<X, B, V, kToken> next;
        if constexpr (kAhead) {
            load_row<X, B, V, kPost, kToken, kAccess>(a, base + team.index * place.rows + place.row,
                                                      end, column, &next);
        }
        float weight[V][N];
        float factor[V][N];  // branch_scale * branch_weight, and the gate unless kToken
        float sum_s[V][N];
        float sum_t[V][N];
        float* lds_t = shares + V * N * static_cast<int>(blockDim.x);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (kLdsSums) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    shares[column[v] + e] = 0.0f;
                    lds_t[column[v] + e] = 0.0f;
                }
            }
            load_weight<kAccess, N>(row_of(a.weight, factor_row(a.weight, begin)), a.weight.dtype,
                                    column[v], a.hidden, weight[v]);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                factor[v][e] = a.branch_scale;
                sum_s[v][e] = 0.0f;
                sum_t[v][e] = 0.0f;
            }
            if constexpr (kPost) {
                float post[N];
                load_weight<kAccess, N>(a.branch_weight, a.branch_weight_dtype, column[v],
                                        a.hidden, post);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    factor[v][e] *= post[e];
                }
            }
            if (!kToken && a.gate.data != nullptr) {
                float gate[N];
                load_weight<kAccess, N>(row_of(a.gate, factor_row(a.gate, begin)), a.gate.dtype,
                                        column[v], a.hidden, gate);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    factor[v][e] *= gate[e];
                }
            }
        }
        for (; base < end; base += step) {
            const int64_t row = base + team.index * place.rows + place.row;
            if constexpr (!kAhead) {
                load_row<X, B, V, kPost, kToken, kAccess>(a, row, end, column, &next);
            }
            Row<X, B, V, kToken> now = next;
            if constexpr (kAhead) {
                if (base + step < end) {
                    load_row<X, B, V, kPost, kToken, kAccess>(a, row + step, end, column, &next);
                }
            }
            const bool live = row < end;
            const int hidden = live ? a.hidden : 0;
            const int64_t first = row * a.hidden;
            const float rstd = now.rstd;
            const float branch_rstd = now.branch_rstd;
            float unit_u[V][N];
            float unit_branch[V][N];
            float gradient[V][N];
            float total[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float gate[N];
                float upstream[N];
                settle<kAccess>(now.u[v], column[v], hidden);
                settle<kAccess>(now.branch[v], column[v], hidden);
                settle<kAccess>(now.grad[v], column[v], hidden);
                widen<X, N>(now.u[v], unit_u[v]);
                widen<B, N>(now.branch[v], unit_branch[v]);
                widen<X, N>(now.grad[v], gradient[v]);
                widen_optional<kAccess, N>(now.upstream[v], a.grad_normalized, a.grad_dtype,
                                           column[v], hidden, 0.0f, upstream);
                if constexpr (kToken && kPost) {
                    widen_any<kAccess, N>(now.gate[v], a.gate.dtype, column[v], hidden, gate);
                }
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    unit_u[v][e] *= rstd;
                    unit_branch[v][e] *= branch_rstd;
                    const float product = upstream[e] * weight[v][e];
                    if constexpr (!kLdsSums) {
                        sum_t[v][e] = __builtin_fmaf(upstream[e], unit_u[v][e], sum_t[v][e]);
                    }
                    gradient[v][e] = __builtin_fmaf(rstd, product, gradient[v][e]);
                    total[0] = __builtin_fmaf(product, unit_u[v][e], total[0]);
                    if constexpr (kPost) {
                        float inner = factor[v][e] * unit_branch[v][e];
                        if constexpr (kToken) {
                            inner *= gate[e];
                        }
                        total[1] = __builtin_fmaf(inner, gradient[v][e], total[1]);
                        total[2] = __builtin_fmaf(inner, unit_u[v][e], total[2]);
                    }
                }
                if constexpr (kLdsSums) {
                    add_products<N>(lds_t + column[v], upstream, unit_u[v]);
                }
            }
            constexpr int kTotals = kPost ? 3 : 1;
#pragma unroll
            for (int i = 0; i < kTotals; ++i) {
                total[i] = row_total<kAccess>(total[i], a.row_lanes);
            }
            if (a.split.parts > 1) {
                // Two buffers: a team's next turn writes the other one while
                // slower waves still read this one.
#pragma unroll
                for (int i = 0; i < kTotals; ++i) {
                    sums[turn][i][team.wave] = total[i];
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kTotals; ++i) {
                    total[i] = 0.0f;
                    for (int part = 0; part < a.split.parts; ++part) {
                        total[i] += sums[turn][i][team.index * a.split.parts + part];
                    }
                }
                turn ^= 1;
            }
            const float shared = rstd * (total[0] * a.inv_hidden);
            const float branch_shared = (total[1] - shared * total[2]) * a.inv_hidden;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float gate[N];
                float grad_x[N];
                float grad_branch[N];
                float each[N];
                if constexpr (kToken) {
                    widen_any<kAccess, N>(now.gate[v], a.gate.dtype, column[v], hidden, gate);
                }
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float g = __builtin_fmaf(-unit_u[v][e], shared, gradient[v][e]);
                    grad_x[e] = a.residual_scale * g;
                    grad_branch[e] = factor[v][e] * g;
                    // A team without a row adds nothing, whatever the factors hold.
                    each[e] = live ? g * unit_branch[v][e] : 0.0f;
                    if constexpr (kToken) {
                        grad_branch[e] *= gate[e];
                    }
                    if constexpr (kPost) {
                        grad_branch[e] = branch_rstd
                            * __builtin_fmaf(-unit_branch[v][e], branch_shared, grad_branch[e]);
                    }
                }
                if constexpr (!kToken) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        gate[e] = 1.0f;
                    }
                }
                if constexpr (kLdsSums) {
                    add_products<N>(shares + column[v], each, gate);
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        sum_s[v][e] = kToken ? __builtin_fmaf(each[e], gate[e], sum_s[v][e])
                                             : sum_s[v][e] + each[e];
                    }
                }
                store<kAccess, kBackwardStores, X, N>(static_cast<X*>(a.grad_x) + first, column[v],
                                                      hidden, narrow<X, N>(grad_x));
                store<kAccess, kBackwardStores, B, N>(static_cast<B*>(a.grad_branch) + first,
                                                      column[v], hidden, narrow<B, N>(grad_branch));
                if (kToken && a.grad_gate != nullptr) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        gate[e] = each[e] * factor[v][e];  // from here on its gradient
                    }
                    store_as<kAccess, kBackwardStores, N>(a.grad_gate, a.gate.dtype, first,
                                                          column[v], hidden, gate);
                }
            }
        }
        if (a.partials == nullptr) {
            continue;
        }
        float* partial = a.partials + unit * 2 * a.hidden;
        if constexpr (kLdsSums) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    sum_s[v][e] = shares[column[v] + e];
                    sum_t[v][e] = lds_t[column[v] + e];
                }
                store<kAccess, kBackwardStores, float, N>(partial, column[v], a.hidden,
                                                          narrow<float, N>(sum_s[v]));
                store<kAccess, kBackwardStores, float, N>(partial + a.hidden, column[v], a.hidden,
                                                          narrow<float, N>(sum_t[v]));
            }
            continue;
        }
        int own[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            own[v] = column[v];
        }
        if constexpr (kAccess == Access::kLanes) {
            // The wave's rows first; row 0's lanes stand for all of them.
#pragma unroll
            for (int e = 0; e < N; ++e) {
                for (int other = a.row_lanes; other < kWave; other *= 2) {
                    sum_s[0][e] += __shfl_xor(sum_s[0][e], other);
                    sum_t[0][e] += __shfl_xor(sum_t[0][e], other);
                }
            }
            if (place.row > 0) {
                own[0] = a.hidden;  // past the end: nothing to leave or to store
            }
        }
        // Teams 1, 2, ... leave their shares; team 0 adds them in that order.
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (team.teams > 1) {
                __syncthreads();  // the shares left before are read
            }
            if (team.index > 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        if (own[v] + e < a.hidden) {
                            shares[(team.index - 1) * a.hidden + own[v] + e] =
                                which == 0 ? sum_s[v][e] : sum_t[v][e];
                        }
                    }
                }
            }
            if (team.teams > 1) {
                __syncthreads();
            }
            if (team.index == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float sum[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        sum[e] = which == 0 ? sum_s[v][e] : sum_t[v][e];
                    }
                    for (int other = 0; other < team.teams - 1; ++other) {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            if (own[v] + e < a.hidden) {
                                sum[e] += shares[other * a.hidden + own[v] + e];
                            }
                        }
                    }
                    store<kAccess, kBackwardStores, float, N>(
                        partial + which * a.hidden, own[v], a.hidden, narrow<float, N>(sum));
                }
            }
        }
    }
}

// ----------------------------------------------------------------------------
// Launch shapes (host). Measured on MI355X, graphs of launches over buffers that pass
// the caches (a large copy reaches 5.1 TB/s there):
//
//  * Forward: two slots of a 16-bit stream, four of a 32-bit one, so that a row has
//    half or a quarter of the waves, which wait for one another twice a row ([6001,
//    2880] bf16 29.7 against 37.8 us with one slot, [16384, 4096] 96 against 101;
//    [8192, 4096] fp32 72.8 against 75.0 with two slots, 116.7 with one). As many blocks
//    of p waves fit a CU as of the next power of two, as measured: 16-bit rows of a
//    normed branch take three slots where that power is less with them ([3640, 4608]
//    29.0 against 41.8 us, [10922, 1536] 27.3 and 29.6, [1364, 12288] 30.4 and 37.7),
//    and not where it is the same ([2340, 7168] 38.9 against 34.1, [2048, 8192] 36.4
//    and 29.4). Branches without a norm wait once a row and show no difference (26.1
//    and 26.3 at 4608); 32-bit rows of six slots are slower ([1820, 4608] 36.1 against
//    31.1). Launches whose waves of one slot are at most half of those that the chip
//    holds take one slot up to 8 waves a row, two beyond: their time is one row's
//    ([512, 4096] bf16 6.0 against 6.5 us, [256, 512] fp32 3.7 against 4.5 with four).
//  * Backward: one slot up to 16 waves a row of a 16-bit stream ([16384, 4096] bf16 155
//    against 192 us with two: the next row's words no longer fit the registers), two
//    from 5 vectors on of a 32-bit one ([4096, 4096] fp32 64 against 74 us, [8192, 1024]
//    37.4 and 37.9).
//  * One block of about 8 waves for each CU, of 9 to 16 where a 16-bit row has 5 waves
//    or more ([16384, 4096] bf16 148 against 162 us, [8192, 2048] 46.7 and 47.8): each block
//    leaves two rows of partial sums, and more blocks cost more in those than they gain
//    ([8192, 4096] fp32 111 against 114 us with two blocks). Two where a block has fewer
//    than 8 waves, and of token gates up to 10, whose next row is not read ahead
//    ([8192, 2048] bf16 62 against 73 us).
//  * Rows of more columns than 16 waves of 8 hold keep their sums in LDS ([2048, 16384]
//    bf16 111-113 us, 154 with sums that left the registers for memory).
//  * A unit's rows are of one group, so groups of fewer rows than a block has teams leave
//    teams idle and nothing to read ahead, and each leaves two rows of partial sums ([8192,
//    4096] bf16 with a weight for each token 733 us, 83 with one for all rows).

inline Split split_of(const Shape& shape) {
    const uint32_t parts = static_cast<uint32_t>(shape.parts);
    return Split{shape.parts, teams_of(shape), ((1u << 16) + parts - 1) / parts};
}

// How a factor's row is found from the stream's: rows / `factor.rows` by the round-up
// method of Granlund and Montgomery (1994), a product with ceil(2^(32 + s) / rows) - 2^32,
// s = ceil(log2(rows)), for 32-bit row numbers.
inline void set_repeat(Factor* factor, int64_t rows) {
    factor->kind = factor->rows >= rows ? kShared
        : factor->rows == 1 ? kToken : rows <= INT32_MAX ? kSample : kWideSample;
    if (factor->kind == kSample) {
        int bits = 1;
        while (int64_t{1} << bits < factor->rows) {
            ++bits;
        }
        const uint64_t divisor = static_cast<uint64_t>(factor->rows);
        factor->magic = static_cast<uint32_t>(
            ((uint64_t{1} << 32) * ((uint64_t{1} << bits) - divisor)) / divisor + 1);
        factor->shift = bits - 1;
    }
}

// `normed`: with a branch weight.
inline Shape pass_shape(int64_t rows, int64_t hidden, int x_dtype, bool normed) {
    if (hidden <= 32 * columns_of(x_dtype)) {
        return short_shape(hidden, x_dtype, 4);
    }
    const int64_t vectors = wave_vectors(hidden, x_dtype);
    const bool resident = rows <= 16 * kComputeUnits && rows * vectors <= 16 * kComputeUnits;
    const int wanted = resident ? (vectors <= 8 ? 1 : 2) : x_dtype == RLN_DTYPE_F32 ? 4 : 2;
    int slots = 1;
    while ((slots < wanted && slots < vectors) || slots * kMaxParts < vectors) {
        slots *= 2;
    }
    const auto held = [&](int of) {  // the next power of two of a row's waves
        int waves = 1;
        while (waves * of < vectors) {
            waves *= 2;
        }
        return waves;
    };
    if (normed && x_dtype != RLN_DTYPE_F32 && slots == 2 && !resident && held(3) < held(2)) {
        slots = 3;  // at most 8 waves: held(2) is at most 16
    }
    return shape_of(vectors, slots, 4);
}

inline Shape walk_shape(int64_t hidden, int x_dtype) {
    if (hidden <= 32 * columns_of(x_dtype)) {
        return short_shape(hidden, x_dtype, 8);
    }
    const int64_t vectors = wave_vectors(hidden, x_dtype);
    int slots = x_dtype == RLN_DTYPE_F32 && vectors > 4 ? 2 : 1;
    while (slots * kMaxParts < vectors) {
        slots *= 2;
    }
    const int waves = x_dtype != RLN_DTYPE_F32 && vectors > 4 && vectors <= kMaxParts ? 12 : 8;
    return shape_of(vectors, slots, waves);
}

// Units of a backward: runs of rows of one group, together at most as many as the
// launch has blocks, but at least one for each group.
struct Units {
    int64_t groups;
    int64_t group_rows;
    int64_t group_units;
    int64_t count;
};

inline Units units_of(int64_t rows, int64_t group_rows, bool token_gate, const Shape& shape) {
    Units units;
    units.group_rows = group_rows;
    units.groups = rows / group_rows;
    const bool two = shape.threads < 8 * kWave || (token_gate && shape.threads <= 10 * kWave);
    const int64_t most = (two ? 2 : 1) * kComputeUnits;
    const int64_t wanted = blocks_of(group_rows, shape);
    const int64_t each = most / units.groups > 0 ? most / units.groups : 1;
    units.group_units = wanted < each ? wanted : each;
    units.count = units.groups * units.group_units;
    return units;
}

// Defined in gated_kernels.hip, one translation unit per stream type and pass.
template <typename X>
int launch_forward(const ForwardArgs& a, const Shape& shape, int branch_dtype, hipStream_t stream);
template <typename X>
int launch_backward(const BackwardArgs& a, const Shape& shape, int branch_dtype,
                    hipStream_t stream);

}  // namespace gated
}  // namespace rln

#endif  // GATED_DEVICE_H
