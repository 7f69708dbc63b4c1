// Rotary positions of query and key heads with the root-mean-square norm of each
// head in front, and their backward (include/rln.h, rln_rotary_*).
//
// Per head h of D values, w its norm's weight:
//
//   n = h * r * w, r = 1 / sqrt(sum(h^2) / D + eps);  without a norm n = h
//   pair i: (n1, n2) -> (n1 cos a - n2 sin a, n1 sin a + n2 cos a), a = p[axis i] * f[i]
//   backward: t the gradient turned by -a, m = t * w,
//             gradient = r * (m - h * r * sum(m * h * r) / D), grad_w = sum of t * h * r
//
// r is taken again from h in the backward: h is read there anyway, and one
// more sum beside sum(m * h) costs less than r's bytes and their allocation.
//
// Bound by memory (4-16 bytes per value against 10-25 operations), as long as the
// angles are not: each is a product in fp64, a reduction to an eighth of a turn and two
// polynomials, about 45 operations, and all heads of a token share them. So a
// block first makes the cosines and sines of a tile of tokens, one pair per thread,
// in LDS, and its lanes then walk the heads of those tokens.
//
// A head belongs to the fewest lanes, a power of two, that hold it: a lane takes two
// vectors of 16 bytes, eight pairs of a 16-bit type (four of fp32): from each half of
// the turned part, or neighbouring ones where pairs are neighbours. Values that are
// not turned follow in vectors of their own, with cosine 1 and sine 0. A wave holds
// 64 / lanes heads, 8 of 128 16-bit values; a sum over a head stays in its lanes.

#include "rms_device.h"

namespace rln {
namespace rotary {
namespace {

using namespace rms;

constexpr int kThreads = 256;
constexpr int64_t kMaxSize = 256;
constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = kMaxSize / 2;

enum class Pass { kTurn, kNorm, kNormBackward };

struct Side {
    const void* heads;
    const void* grad;   // the backward's
    const void* weight;
    void* output;
    int64_t heads_outer, heads_token, heads_head;
    int64_t grad_outer, grad_token, grad_head;
    int count;
    float inverse_count;
    int weight_dtype;
};

struct Args {
    Side side[2];
    const void* positions;
    const void* frequencies;
    float* partials;          // [blocks][2][size], or null
    int64_t position_axis, position_outer, position_token;
    int tokens;
    int inner;
    int tile;                 // tokens
    int tiles;
    int size;
    int pairs;
    int row_pairs;            // of a token in LDS: pairs in whole vectors
    float inverse_row_pairs;
    int lanes;                // of a head
    int turned_lanes;         // those of turned values
    int positions_type;
    int wide_frequencies;
    int interleaved;
    int backward;             // angles are taken negative
    float eps;
    float inverse_size;
    uint32_t axes[kMaxPairs / 16];  // 2 bits per pair
};

// ----------------------------------------------------------------------------
// Angles.

__device__ __forceinline__ double position_of(const Args& a, int axis, int token) {
    int64_t offset = axis * a.position_axis;
    if (a.inner < a.tokens) {
        const int outer = token / a.inner;
        offset += outer * a.position_outer + (token - outer * a.inner) * a.position_token;
    } else {
        offset += token * a.position_token;
    }
    switch (a.positions_type) {
        case RLN_POSITIONS_I64:
            return static_cast<double>(static_cast<const int64_t*>(a.positions)[offset]);
        case RLN_POSITIONS_I32:
            return static_cast<double>(static_cast<const int32_t*>(a.positions)[offset]);
        default:
            return static_cast<double>(static_cast<const float*>(a.positions)[offset]);
    }
}

// Cosine and sine, each within about one unit in the last place: whole quarters of
// a turn are taken off in fp64, by pi / 2 in two parts, so that far angles lose nothing
// but their own rounding; the rest, at most an eighth of a turn, goes into the Taylor
// polynomials (their first omitted terms are below 2^-24 of the value there).
__device__ __forceinline__ void turn_of(double angle, float* cosine, float* sine) {
    const double whole = __builtin_rint(angle * 0.6366197723675814);  // 2 / pi
    const double near = __builtin_fma(-whole, 1.5707963267948966, angle);
    const float x = static_cast<float>(__builtin_fma(-whole, 6.123233995736766e-17, near));
    const float x2 = x * x;
    float s = __builtin_fmaf(x2, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = __builtin_fmaf(x2, s, 1.0f / 120.0f);
    s = __builtin_fmaf(x2, s, -1.0f / 6.0f);
    s = __builtin_fmaf(x2 * x, s, x);
    float c = __builtin_fmaf(x2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = __builtin_fmaf(x2, c, -1.0f / 720.0f);
    c = __builtin_fmaf(x2, c, 1.0f / 24.0f);
    c = __builtin_fmaf(x2, c, -0.5f);
    c = __builtin_fmaf(x2, c, 1.0f);
    const int quadrant =
        static_cast<int>(__builtin_fma(-4.0, __builtin_rint(whole * 0.25), whole)) & 3;
    const float swapped_s = quadrant & 1 ? c : s;
    const float swapped_c = quadrant & 1 ? s : c;
    *sine = quadrant & 2 ? -swapped_s : swapped_s;
    *cosine = (quadrant + 1) & 2 ? -swapped_c : swapped_c;
}

// ----------------------------------------------------------------------------
// A lane's two vectors of a head.

struct Place {
    int base[2];    // the first element of the run that a vector belongs to
    int column[2];  // the vector's first element in it
    int extent;     // the run's elements (0: no vector)
    int pair;       // the lane's first pair, or -1 where nothing is turned
};

template <int N>
__device__ __forceinline__ Place place_of(const Args& a, int chunk) {
    Place place;
    const int turned = 2 * a.pairs;
    place.pair = -1;
    if (chunk < a.turned_lanes) {
        place.pair = chunk * N;
        place.base[0] = 0;
        place.base[1] = a.interleaved ? 0 : a.pairs;
        place.column[0] = a.interleaved ? 2 * N * chunk : N * chunk;
        place.column[1] = a.interleaved ? 2 * N * chunk + N : N * chunk;
        place.extent = a.interleaved ? turned : a.pairs;
    } else {
        place.base[0] = place.base[1] = turned;
        place.column[0] = 2 * N * (chunk - a.turned_lanes);
        place.column[1] = place.column[0] + N;
        place.extent = a.size - turned;
    }
    return place;
}

// kWhole: every run is whole vectors, so that one is read or not at all.
template <bool kWhole, typename T, int N>
__device__ __forceinline__ Raw<T, N> load_vector(const T* head, const Place& place, int half,
                                                 bool live) {
    const T* run = head + place.base[half];
    const int extent = live ? place.extent : 0;
    if constexpr (kWhole) {
        using W = WordVector<4, static_cast<int>(sizeof(T))>;
        typename W::plain words{};
        if (place.column[half] < extent) {
            words = __builtin_nontemporal_load(
                reinterpret_cast<const typename W::type*>(run + place.column[half]));
        }
        Raw<T, N> raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            raw.words[i] = words[i];
        }
        return raw;
    } else {
        return load<Access::kLanes, T, N>(run, place.column[half], extent);
    }
}

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void widen_vector(Raw<T, N>& raw, const Place& place, int half,
                                             bool live, float (&out)[N]) {
    if constexpr (!kWhole) {
        settle<Access::kLanes>(raw, place.column[half], live ? place.extent : 0);
    }
    widen<T, N>(raw, out);
}

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void store_vector(T* head, const Place& place, int half,
                                             const float (&values)[N]) {
    T* run = head + place.base[half];
    if constexpr (kWhole) {
        if (place.column[half] < place.extent) {
            const Raw<T, N> raw = narrow<T, N>(values);
            using W = WordVector<4, static_cast<int>(sizeof(T))>;
            const typename W::plain words = {raw.words[0], raw.words[1], raw.words[2],
                                             raw.words[3]};
            __builtin_nontemporal_store(
                words, reinterpret_cast<typename W::type*>(run + place.column[half]));
        }
    } else {
        store<Access::kLanes, kForwardStores, T, N>(run, place.column[half], place.extent,
                                                    narrow<T, N>(values));
    }
}

template <int N>
__device__ __forceinline__ void read_lds(const float* from, float (&out)[N]) {
    typedef float Four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const Four four = *reinterpret_cast<const Four*>(from + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            out[i + k] = four[k];
        }
    }
}

template <int N>
__device__ __forceinline__ void turn(float (&first)[N], float (&second)[N],
                                     const float (&cosine)[N], const float (&sine)[N],
                                     bool interleaved) {
    const auto pair = [](float& x, float& y, float c, float s) {
        const float turned = x * c - y * s;
        y = x * s + y * c;
        x = turned;
    };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            pair(first[2 * i], first[2 * i + 1], cosine[i], sine[i]);
            pair(second[2 * i], second[2 * i + 1], cosine[N / 2 + i], sine[N / 2 + i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            pair(first[i], second[i], cosine[i], sine[i]);
        }
    }
}

// Sum over each aligned run of `lanes` lanes, a power of two.
__device__ __forceinline__ float head_sum(float value, int lanes) {
#define ROTARY_ADD(control) \
    value += __builtin_bit_cast(float, RMS_DPP(__builtin_bit_cast(uint32_t, value), control))
    if (lanes > 1) {
        ROTARY_ADD(kXor1);
    }
    if (lanes > 2) {
        ROTARY_ADD(kXor2);
    }
    if (lanes > 4) {
        ROTARY_ADD(kHalfMirror);
    }
    if (lanes > 8) {
        ROTARY_ADD(kMirror);
    }
#undef ROTARY_ADD
    if (lanes > 16) {
        value += __shfl_xor(value, 16);
    }
    if (lanes > 32) {
        value += __shfl_xor(value, 32);
    }
    return value;
}

// ----------------------------------------------------------------------------
// One block per tile of tokens and share of their heads (blockIdx.y); in the
// backward with a norm the blocks walk the tiles, so that a block leaves one row of
// partial sums, which reduce_kernel adds in a fixed order.

template <typename T, Pass kPass, bool kWhole>
__global__ __launch_bounds__(kThreads) void heads_kernel(Args a) {
    constexpr int N = kColumns<T>;
    constexpr bool kNormed = kPass != Pass::kTurn;
    constexpr bool kSums = kPass == Pass::kNormBackward;
    // Cosines and sines [tile][row_pairs] each, then the weights [2][lanes][2][N].
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int angles = a.tile * a.row_pairs;
    float* cosines = lds;
    float* sines = lds + angles;
    float* weights = lds + 2 * angles;
    const int chunk = static_cast<int>(threadIdx.x) % a.lanes;
    const int slot = static_cast<int>(threadIdx.x) / a.lanes;
    const int slots = kThreads / a.lanes;
    const Place place = place_of<N>(a, chunk);
    if constexpr (kNormed) {
        for (int i = static_cast<int>(threadIdx.x); i < 4 * a.lanes; i += kThreads) {
            const int half = i & 1;
            const Place at = place_of<N>(a, (i >> 1) % a.lanes);
            const Side& side = a.side[(i >> 1) / a.lanes];
            float values[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int column = at.column[half] + e;
                const int64_t index = at.base[half] + column;
                values[e] = 0.0f;
                if (side.weight != nullptr && column < at.extent) {
                    values[e] = side.weight_dtype == RLN_DTYPE_F32
                        ? static_cast<const float*>(side.weight)[index]
                        : side.weight_dtype == RLN_DTYPE_F16
                        ? static_cast<float>(static_cast<const half_t*>(side.weight)[index])
                        : static_cast<float>(static_cast<const bf16_t*>(side.weight)[index]);
                }
                weights[i * N + e] = values[e];
            }
        }
    }
    float sums[2][2][N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
        (&sums[0][0][0])[i] = 0.0f;
    }
    for (int tile = static_cast<int>(blockIdx.x); tile < a.tiles;
         tile += static_cast<int>(gridDim.x)) {
        const int begin = tile * a.tile;
        const int tokens = a.tokens - begin < a.tile ? a.tokens - begin : a.tile;
        for (int i = static_cast<int>(threadIdx.x); i < tokens * a.row_pairs; i += kThreads) {
            const int token =
                static_cast<int>((static_cast<float>(i) + 0.5f) * a.inverse_row_pairs);
            const int pair = i - token * a.row_pairs;
            float cosine = 1.0f;
            float sine = 0.0f;
            if (pair < a.pairs) {
                const int axis = static_cast<int>(a.axes[pair >> 4] >> (2 * (pair & 15)) & 3u);
                const double frequency = a.wide_frequencies
                    ? static_cast<const double*>(a.frequencies)[pair]
                    : static_cast<double>(static_cast<const float*>(a.frequencies)[pair]);
                turn_of(position_of(a, axis, begin + token) * frequency, &cosine, &sine);
            }
            cosines[i] = cosine;
            sines[i] = a.backward ? -sine : sine;
        }
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const Side& side = a.side[which];
            const bool normed = kNormed && side.weight != nullptr;
            float weight[2][N];
            if constexpr (kNormed) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    read_lds<N>(weights + ((which * a.lanes + chunk) * 2 + half) * N,
                                weight[half]);
                }
            }
            const int rows = tokens * side.count;
            for (int row = slot + static_cast<int>(blockIdx.y) * slots; row < rows;
                 row += slots * static_cast<int>(gridDim.y)) {
                const int local =
                    static_cast<int>((static_cast<float>(row) + 0.5f) * side.inverse_count);
                const int head = row - local * side.count;
                const int token = begin + local;
                int outer = 0;
                int within = token;
                if (a.inner < a.tokens) {
                    outer = token / a.inner;
                    within = token - outer * a.inner;
                }
                // What is turned: the heads, or the backward's gradient.
                const bool back = a.backward != 0;
                const T* from = back
                    ? static_cast<const T*>(side.grad) + outer * side.grad_outer
                        + within * side.grad_token + head * side.grad_head
                    : static_cast<const T*>(side.heads) + outer * side.heads_outer
                        + within * side.heads_token + head * side.heads_head;
                Raw<T, N> raw[2];
                Raw<T, N> raw_heads[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    raw[half] = load_vector<kWhole, T, N>(from, place, half, true);
                }
                if constexpr (kSums) {
                    const T* heads = static_cast<const T*>(side.heads)
                        + outer * side.heads_outer + within * side.heads_token
                        + head * side.heads_head;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        raw_heads[half] = load_vector<kWhole, T, N>(heads, place, half, normed);
                    }
                }
                float values[2][N];
                float cosine[N];
                float sine[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    cosine[e] = 1.0f;
                    sine[e] = 0.0f;
                }
                if (place.pair >= 0) {
                    read_lds<N>(cosines + local * a.row_pairs + place.pair, cosine);
                    read_lds<N>(sines + local * a.row_pairs + place.pair, sine);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    widen_vector<kWhole, T, N>(raw[half], place, half, true, values[half]);
                }
                if constexpr (kPass == Pass::kNorm) {
                    if (normed) {
                        float sum = 0.0f;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                sum += values[half][e] * values[half][e];
                            }
                        }
                        sum = head_sum(sum, a.lanes);
                        const float rstd =
                            1.0f / __builtin_sqrtf(sum * a.inverse_size + a.eps);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                values[half][e] *= rstd * weight[half][e];
                            }
                        }
                    }
                }
                turn<N>(values[0], values[1], cosine, sine, a.interleaved != 0);
                if constexpr (kSums) {
                    if (normed) {
                        float unit[2][N];
                        float square = 0.0f;
                        float shared = 0.0f;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            widen_vector<kWhole, T, N>(raw_heads[half], place, half, normed,
                                                       unit[half]);
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                square += unit[half][e] * unit[half][e];
                                shared += values[half][e] * weight[half][e] * unit[half][e];
                            }
                        }
                        square = head_sum(square, a.lanes);
                        shared = head_sum(shared, a.lanes);
                        const float rstd =
                            1.0f / __builtin_sqrtf(square * a.inverse_size + a.eps);
                        shared *= rstd * a.inverse_size;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                const float normal = unit[half][e] * rstd;
                                sums[which][half][e] += values[half][e] * normal;
                                values[half][e] = rstd
                                    * (values[half][e] * weight[half][e] - normal * shared);
                            }
                        }
                    }
                }
                T* to = static_cast<T*>(side.output)
                    + (static_cast<int64_t>(token) * side.count + head) * a.size;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    store_vector<kWhole, T, N>(to, place, half, values[half]);
                }
            }
        }
        __syncthreads();  // the tile's angles are read before the next one's are written
    }
    if constexpr (kSums) {
        if (a.partials == nullptr) {
            return;
        }
        // The wave's heads by exchanges, the block's waves through LDS, in their order.
        constexpr int kWaves = kThreads / kWave;
        const int wave = static_cast<int>(threadIdx.x) / kWave;
        const int lane = static_cast<int>(threadIdx.x) % kWave;
        const int vectors = 4 * a.lanes;  // [2][lanes][2] of N
#pragma unroll
        for (int which = 0; which < 2; ++which) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    float sum = sums[which][half][e];
                    for (int other = a.lanes; other < kWave; other *= 2) {
                        sum += __shfl_xor(sum, other);
                    }
                    if (lane < a.lanes) {
                        lds[(wave * vectors + (which * a.lanes + chunk) * 2 + half) * N + e] = sum;
                    }
                }
            }
        }
        __syncthreads();
        float* partial = a.partials
            + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * a.size;
        for (int i = static_cast<int>(threadIdx.x); i < vectors * N; i += kThreads) {
            const int e = i % N;
            const int vector = i / N;
            const int half = vector & 1;
            const Place at = place_of<N>(a, (vector >> 1) % a.lanes);
            const int which = (vector >> 1) / a.lanes;
            if (at.column[half] + e < at.extent) {
                float sum = lds[i];
                for (int other = 1; other < kWaves; ++other) {
                    sum += lds[other * vectors * N + i];
                }
                partial[which * a.size + at.base[half] + at.column[half] + e] = sum;
            }
        }
    }
}

// Fixed-order sums of the partials [blocks][2][size], rounded once to the weights'
// types. A block owns 16 columns; its 64 groups of 16 lanes take every 64th row.
constexpr int kReduceColumns = 16;
constexpr int kReduceGroups = 64;

struct ReduceArgs {
    const float* partials;
    void* grad_weight[2];
    int dtype[2];
    int blocks;
    int size;
};

__global__ __launch_bounds__(kReduceColumns * kReduceGroups) void reduce_kernel(ReduceArgs a) {
    __shared__ float totals[kReduceGroups][kReduceColumns + 1];
    const int which = blockIdx.y;
    if (a.grad_weight[which] == nullptr) {
        return;
    }
    const int lane = threadIdx.x % kReduceColumns;
    const int group = threadIdx.x / kReduceColumns;
    const int column = blockIdx.x * kReduceColumns + lane;
    float total = 0.0f;
    if (column < a.size) {
#pragma unroll 8
        for (int block = group; block < a.blocks; block += kReduceGroups) {
            total += a.partials[(static_cast<int64_t>(block) * 2 + which) * a.size + column];
        }
    }
    totals[group][lane] = total;
    __syncthreads();
    if (group == 0 && column < a.size) {
        for (int other = 1; other < kReduceGroups; ++other) {
            total += totals[other][lane];
        }
        store_one(a.grad_weight[which], a.dtype[which], column, total);
    }
}

// ----------------------------------------------------------------------------
// Launch shapes and checks (host).

struct Grid {
    int lanes;
    int turned_lanes;
    int tile;
    int tiles;
    int row_pairs;
    unsigned x;
    unsigned y;
    bool whole;
};

// A tile has about as many pairs as the block has threads, so that each makes one
// angle, and a launch of few tokens spreads their heads over more blocks. A backward
// with sums walks its tiles with at most four blocks for each CU.
Grid grid_of(int64_t tokens, int64_t most_heads, int64_t size, int64_t pairs, int dtype,
             bool sums) {
    Grid grid;
    const int columns = columns_of(dtype);
    const int left = static_cast<int>(size - 2 * pairs);
    grid.turned_lanes = static_cast<int>((pairs + columns - 1) / columns);
    const int vectors = grid.turned_lanes + (left + 2 * columns - 1) / (2 * columns);
    grid.lanes = 1;
    while (grid.lanes < vectors) {
        grid.lanes *= 2;
    }
    grid.row_pairs = grid.turned_lanes * columns;
    grid.whole = pairs % columns == 0 && left % (2 * columns) == 0;
    const int full = kThreads / (grid.row_pairs > 0 ? grid.row_pairs : 1);
    grid.tile = full < 1 ? 1 : full > 16 ? 16 : full;
    while (grid.tile > 1 && tokens / grid.tile < 4 * kComputeUnits) {
        grid.tile /= 2;
    }
    grid.tiles = static_cast<int>((tokens + grid.tile - 1) / grid.tile);
    const int slots = kThreads / grid.lanes;
    const int64_t passes = (grid.tile * most_heads + slots - 1) / slots;
    const int64_t wanted = 4 * kComputeUnits;
    const int64_t share = wanted / grid.tiles > 1 ? wanted / grid.tiles : 1;
    grid.y = static_cast<unsigned>(passes < share ? passes : share);
    grid.x = static_cast<unsigned>(sums && grid.tiles > wanted ? wanted : grid.tiles);
    return grid;
}

bool float_dtype(int dtype) {
    return dtype == RLN_DTYPE_F32 || dtype == RLN_DTYPE_F16 || dtype == RLN_DTYPE_BF16;
}

int64_t size_of(int dtype) {
    return dtype == RLN_DTYPE_F32 ? 4 : 2;
}

int check_address(const char* name, const void* data, int64_t bytes) {
    if (reinterpret_cast<uintptr_t>(data) % bytes != 0) {
        return fail(RLN_ERR_INVALID, "%s is not aligned to its elements", name);
    }
    return RLN_OK;
}

// Strides whose farthest element's offset fits int64.
int check_strides(const char* name, const int64_t (&strides)[3], const int64_t (&counts)[3]) {
    for (int i = 0; i < 3; ++i) {
        const int64_t limit = INT64_MAX / 64 / (counts[i] > 1 ? counts[i] : 1);
        if (strides[i] > limit || strides[i] < -limit) {
            return fail(RLN_ERR_INVALID, "%s: the strides overflow int64", name);
        }
    }
    return RLN_OK;
}

int check_heads(const char* name, const rln_heads_t& heads, int dtype, int64_t outer,
                int64_t inner, int64_t count) {
    if (heads.data == nullptr) {
        return fail(RLN_ERR_INVALID, "%s must not be null", name);
    }
    const int64_t strides[3] = {heads.outer_stride, heads.token_stride, heads.head_stride};
    const int64_t counts[3] = {outer, inner, count};
    const int status = check_strides(name, strides, counts);
    return status != RLN_OK ? status : check_address(name, heads.data, size_of(dtype));
}

int check_side(const char* name, const rln_rotary_side_t* given, int dtype, int64_t outer,
               int64_t inner, int64_t size, bool backward, Side* side) {
    *side = Side{};
    if (given == nullptr || given->count == 0) {
        return RLN_OK;
    }
    // The rows of a tile of 16 tokens are divided by the count in fp32.
    if (given->count < 0 || given->count > 1 << 16) {
        return fail(RLN_ERR_UNSUPPORTED, "%s: unsupported number of heads: %lld", name,
                    static_cast<long long>(given->count));
    }
    if (outer * inner > INT64_MAX / 8 / (given->count * size)) {
        return fail(RLN_ERR_INVALID, "%s: its elements overflow int64", name);
    }
    int status = RLN_OK;
    const bool reads_heads = !backward || given->weight != nullptr;
    if ((reads_heads
         && (status = check_heads(name, given->heads, dtype, outer, inner, given->count))
             != RLN_OK)
        || (backward
            && (status = check_heads("grad", given->grad, dtype, outer, inner, given->count))
                != RLN_OK)) {
        return status;
    }
    if (given->output == nullptr) {
        return fail(RLN_ERR_INVALID, "%s: output must not be null", name);
    }
    if ((status = check_address("output", given->output, size_of(dtype))) != RLN_OK) {
        return status;
    }
    if (given->weight != nullptr) {
        if (!float_dtype(given->weight_dtype)) {
            return fail(RLN_ERR_INVALID, "weight must use float16, bfloat16 or float32");
        }
        if ((status = check_address("weight", given->weight, size_of(given->weight_dtype)))
            != RLN_OK) {
            return status;
        }
    }
    if (given->grad_weight != nullptr) {
        if (!backward || given->weight == nullptr) {
            return fail(RLN_ERR_INVALID, "grad_weight without a weight");
        }
        if ((status = check_address("grad_weight", given->grad_weight,
                                    size_of(given->weight_dtype))) != RLN_OK) {
            return status;
        }
    }
    side->heads = given->heads.data;
    side->heads_outer = given->heads.outer_stride;
    side->heads_token = given->heads.token_stride;
    side->heads_head = given->heads.head_stride;
    side->grad = given->grad.data;
    side->grad_outer = given->grad.outer_stride;
    side->grad_token = given->grad.token_stride;
    side->grad_head = given->grad.head_stride;
    side->weight = given->weight;
    side->weight_dtype = given->weight_dtype;
    side->output = given->output;
    side->count = static_cast<int>(given->count);
    side->inverse_count = 1.0f / static_cast<float>(given->count);
    return RLN_OK;
}

int check_rotary(const rln_rotary_t* given, int64_t outer, int64_t inner, int64_t size, Args* a) {
    if (given == nullptr || given->positions == nullptr || given->frequencies == nullptr) {
        return fail(RLN_ERR_INVALID, "positions and frequencies must not be null");
    }
    if (given->pairs < 1 || 2 * given->pairs > size) {
        return fail(RLN_ERR_INVALID, "the pairs must be 1 to half of the head's size");
    }
    if (given->axes < 1 || given->axes > kMaxAxes) {
        return fail(RLN_ERR_INVALID, "positions must have 1 to 4 axes");
    }
    if (given->positions_type != RLN_POSITIONS_I64 && given->positions_type != RLN_POSITIONS_I32
        && given->positions_type != RLN_POSITIONS_F32) {
        return fail(RLN_ERR_INVALID, "positions must use int64, int32 or float32");
    }
    int status = check_address("positions", given->positions,
                               given->positions_type == RLN_POSITIONS_I64 ? 8 : 4);
    if (status != RLN_OK
        || (status = check_address("frequencies", given->frequencies,
                                   given->wide_frequencies ? 8 : 4)) != RLN_OK) {
        return status;
    }
    const int64_t strides[3] = {given->axis_stride, given->outer_stride, given->token_stride};
    const int64_t counts[3] = {given->axes, outer, inner};
    if ((status = check_strides("positions", strides, counts)) != RLN_OK) {
        return status;
    }
    if (given->axis_of_pair != nullptr) {
        for (int64_t pair = 0; pair < given->pairs; ++pair) {
            if (given->axis_of_pair[pair] >= given->axes) {
                return fail(RLN_ERR_INVALID, "axis_of_pair holds an axis past the last");
            }
            a->axes[pair / 16] |= static_cast<uint32_t>(given->axis_of_pair[pair])
                << (2 * (pair % 16));
        }
    }
    a->positions = given->positions;
    a->positions_type = given->positions_type;
    a->position_axis = given->axis_stride;
    a->position_outer = given->outer_stride;
    a->position_token = given->token_stride;
    a->frequencies = given->frequencies;
    a->wide_frequencies = given->wide_frequencies;
    a->pairs = static_cast<int>(given->pairs);
    a->interleaved = given->interleaved;
    return RLN_OK;
}

// Everything but the launch; `grid` receives its shape.
int arguments(const rln_rotary_side_t* q, const rln_rotary_side_t* k, int dtype,
              const rln_rotary_t* rotary, int64_t outer, int64_t inner, int64_t size, double eps,
              void* stream, bool backward, Args* a, Grid* grid, bool* normed) {
    if (!float_dtype(dtype)) {
        return fail(RLN_ERR_INVALID, "heads must use float16, bfloat16 or float32");
    }
    if (outer < 1 || inner < 1) {
        return fail(RLN_ERR_INVALID, "empty tensors are unsupported");
    }
    if (inner > INT32_MAX / 2 || outer > INT32_MAX / 2 / inner) {
        return fail(RLN_ERR_UNSUPPORTED, "unsupported number of tokens");
    }
    if (size < 1 || size > kMaxSize) {
        return fail(RLN_ERR_UNSUPPORTED, "unsupported head size: %lld",
                    static_cast<long long>(size));
    }
    if (!(eps >= 0.0)) {
        return fail(RLN_ERR_INVALID, "eps must not be negative");
    }
    *a = Args{};
    int status = check_rotary(rotary, outer, inner, size, a);
    if (status != RLN_OK
        || (status = check_side("q", q, dtype, outer, inner, size, backward, &a->side[0]))
            != RLN_OK
        || (status = check_side("k", k, dtype, outer, inner, size, backward, &a->side[1]))
            != RLN_OK) {
        return status;
    }
    const int most = a->side[0].count > a->side[1].count ? a->side[0].count : a->side[1].count;
    if (most == 0) {
        return fail(RLN_ERR_INVALID, "empty tensors are unsupported");
    }
    if ((status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    *normed = a->side[0].weight != nullptr || a->side[1].weight != nullptr;
    *grid = grid_of(outer * inner, most, size, a->pairs, dtype, backward && *normed);
    a->tokens = static_cast<int>(outer * inner);
    a->inner = static_cast<int>(inner);
    a->tile = grid->tile;
    a->tiles = grid->tiles;
    a->size = static_cast<int>(size);
    a->row_pairs = grid->row_pairs;
    a->inverse_row_pairs = 1.0f / static_cast<float>(grid->row_pairs);
    a->lanes = grid->lanes;
    a->turned_lanes = grid->turned_lanes;
    a->backward = backward;
    a->eps = static_cast<float>(eps);
    a->inverse_size = 1.0f / static_cast<float>(size);
    return RLN_OK;
}

template <typename T, Pass kPass>
int launch(const Args& a, const Grid& grid, hipStream_t stream) {
    const size_t weights = kPass == Pass::kTurn ? 0 : 4 * a.lanes * kColumns<T>;
    size_t floats = 2 * static_cast<size_t>(a.tile) * a.row_pairs + weights;
    if (kPass == Pass::kNormBackward && floats < kThreads / kWave * weights) {
        floats = kThreads / kWave * weights;  // the block's sums, in the same place
    }
    const auto kernel =
        grid.whole ? heads_kernel<T, kPass, true> : heads_kernel<T, kPass, false>;
    kernel<<<dim3(grid.x, grid.y), kThreads, floats * sizeof(float), stream>>>(a);
    return check_launch("rotary heads_kernel");
}

template <typename T>
int launch_pass(const Args& a, const Grid& grid, bool normed, hipStream_t stream) {
    if (!normed) {
        return launch<T, Pass::kTurn>(a, grid, stream);
    }
    return a.backward ? launch<T, Pass::kNormBackward>(a, grid, stream)
                      : launch<T, Pass::kNorm>(a, grid, stream);
}

int launch_dtype(const Args& a, const Grid& grid, int dtype, bool normed, void* stream) {
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RLN_DTYPE_F32:
            return launch_pass<float>(a, grid, normed, queue);
        case RLN_DTYPE_F16:
            return launch_pass<half_t>(a, grid, normed, queue);
        default:
            return launch_pass<bf16_t>(a, grid, normed, queue);
    }
}

}  // namespace
}  // namespace rotary
}  // namespace rln

using namespace rln;
using namespace rln::rotary;

extern "C" {

int rln_rotary_forward(
    const rln_rotary_side_t* q, const rln_rotary_side_t* k, int dtype,
    const rln_rotary_t* rotary, int64_t outer, int64_t inner, int64_t size, double eps,
    void* stream) {
    clear_error();
    Args a;
    Grid grid;
    bool normed = false;
    const int status = arguments(q, k, dtype, rotary, outer, inner, size, eps, stream, false, &a,
                                 &grid, &normed);
    return status != RLN_OK ? status : launch_dtype(a, grid, dtype, normed, stream);
}

size_t rln_rotary_backward_workspace_bytes(
    int64_t outer, int64_t inner, int64_t q_heads, int64_t k_heads, int64_t size, int64_t pairs,
    int dtype) {
    const int64_t most = q_heads > k_heads ? q_heads : k_heads;
    if (!float_dtype(dtype) || outer < 1 || inner < 1 || inner > INT32_MAX / 2
        || outer > INT32_MAX / 2 / inner || size < 1 || size > kMaxSize || pairs < 1
        || 2 * pairs > size || most < 1 || most > 1 << 16) {
        return 0;
    }
    const Grid grid = grid_of(outer * inner, most, size, pairs, dtype, true);
    return static_cast<size_t>(grid.x) * grid.y * 2 * static_cast<size_t>(size) * sizeof(float);
}

int rln_rotary_backward(
    const rln_rotary_side_t* q, const rln_rotary_side_t* k, int dtype,
    const rln_rotary_t* rotary, int64_t outer, int64_t inner, int64_t size, double eps,
    void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    Args a;
    Grid grid;
    bool normed = false;
    int status = arguments(q, k, dtype, rotary, outer, inner, size, eps, stream, true, &a, &grid,
                           &normed);
    if (status != RLN_OK) {
        return status;
    }
    ReduceArgs reduce{};
    reduce.grad_weight[0] = a.side[0].count > 0 ? q->grad_weight : nullptr;
    reduce.grad_weight[1] = a.side[1].count > 0 ? k->grad_weight : nullptr;
    const bool sums = reduce.grad_weight[0] != nullptr || reduce.grad_weight[1] != nullptr;
    if (sums) {
        const size_t needed =
            static_cast<size_t>(grid.x) * grid.y * 2 * static_cast<size_t>(size) * sizeof(float);
        if (workspace == nullptr || workspace_bytes < needed) {
            return fail(RLN_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", needed,
                        workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
        }
        if ((status = check_address("workspace", workspace, 4)) != RLN_OK) {
            return status;
        }
        a.partials = static_cast<float*>(workspace);
    }
    status = launch_dtype(a, grid, dtype, normed, stream);
    if (status != RLN_OK || !sums) {
        return status;
    }
    reduce.partials = a.partials;
    reduce.dtype[0] = a.side[0].weight_dtype;
    reduce.dtype[1] = a.side[1].weight_dtype;
    reduce.blocks = static_cast<int>(grid.x * grid.y);
    reduce.size = a.size;
    const unsigned blocks = static_cast<unsigned>((size + kReduceColumns - 1) / kReduceColumns);
    reduce_kernel<<<dim3(blocks, 2), kReduceColumns * kReduceGroups, 0,
                    static_cast<hipStream_t>(stream)>>>(reduce);
    return check_launch("rotary reduce_kernel");
}

}  // extern "C"
