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
// block first makes the cosines and sines of a tile of tokens in LDS, and its lanes then
// walk the heads of those tokens, those of q or those of k: one side's weight and sums
// fit the registers beside a head that is read ahead. Turns without a norm have neither
// and take the same blocks, which make their angles for each side ([6001, 28 + 4 heads
// of 128] bf16 24 us; a simpler kernel with blocks of both sides took 22).
//
// A head belongs to the fewest lanes, a power of two, that hold it: a lane takes two
// vectors of 16 bytes, eight pairs of a 16-bit type (four of fp32): from each half of
// the turned part, or neighbouring ones where pairs are neighbours. Values that are
// not turned follow in vectors of their own, in lanes that turn nothing. A wave holds
// 64 / lanes heads, 8 of 128 16-bit values; a sum over a head stays in its lanes, and
// a lane's columns, hence its weights, are the same for every head it walks.
//
// Measured: [16384, 32 + 8 heads of 128] bf16 with norms, forward 67 us, backward 100,
// both 5.0 TB/s, what a large copy reaches (in graphs 70 and 115 where 4 samples share
// positions, 72 and 119 with heads before tokens, 69 and 113 as one run); [8192, 12 + 12
// of 64] fp16 15.5 and 25.4 (3.0-3.2 TB/s: the halves of such a head fill half a line
// each); [8858, 16 + 16 of 72] fp16 24-28 (9 lanes of 16 hold a head); 16 tokens of 32 +
// 8 of 128 3.8.

#include "rms_device.h"

namespace rln {
namespace rotary {
namespace {

using namespace rms;

constexpr int kThreads = 256;
constexpr int64_t kMaxSize = 256;
constexpr int kMaxAxes = 4;
constexpr int64_t kMaxHeads = 1 << 16;
constexpr int kMaxPairs = kMaxSize / 2;
constexpr int kTilePairs = 2048;  // 16 KB of LDS

enum class Pass { kTurn, kNorm, kNormBackward };

struct Side {
    const void* heads;  // what is turned; in a backward with a norm, its heads
    const void* grad;   // and what is turned there
    const void* weight;
    void* output;
    float* partials;    // [blocks][size], or null
    int64_t heads_outer, heads_token, heads_head;
    int64_t grad_outer, grad_token, grad_head;
    // From a head to the one that a lane takes next, row_step heads on: tokens and heads,
    // and elements of both tensors, the latter for a token more and `count` heads less.
    int step_tokens, step_heads;
    int64_t heads_step, heads_wrap;
    int64_t grad_step, grad_wrap;
    int row_step;
    int count;
    float inverse_count;
    int weight_dtype;
    int tile;           // tokens
    int parts;          // blocks that share a tile's heads
    int items;          // tiles * parts
    int blocks;         // which walk the items
};

struct Args {
    Side side[2];             // the launch's first side[0].blocks are q's
    const void* positions;
    const void* frequencies;
    int64_t position_axis, position_outer, position_token;
    int tokens;
    int inner;
    int size;
    int pairs;
    int row_pairs;            // of a token in LDS: pairs in whole vectors
    float inverse_row_pairs;
    int lanes;                // of a head
    int lanes_shift;
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

// kWhole: every run is whole vectors, so that one is read or not at all. Cached loads:
// a head's half is less than a line where heads are short, and its line is read twice
// ([8192, 24 heads of 64] fp16 13.9 us, 16.5 with loads that do not stay; longer heads the
// same); the outputs are not read here and do not stay ([16384, 40 of 128] bf16 69
// against 73 us with plain stores).
template <bool kWhole, typename T, int N>
__device__ __forceinline__ Raw<T, N> load_vector(const T* head, const Place& place, int half,
                                                 int extent) {
    const T* run = head + place.base[half];
    if constexpr (kWhole) {
        constexpr int kWords = Raw<T, N>::kWords;
        using W = WordVector<kWords, static_cast<int>(sizeof(T))>;
        typename W::plain words{};
        if (place.column[half] < extent) {
            words = *reinterpret_cast<const typename W::type*>(run + place.column[half]);
        }
        Raw<T, N> raw;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            raw.words[i] = words[i];
        }
        return raw;
    } else {
        return load<Access::kLanes, T, N, kCached>(run, place.column[half], extent);
    }
}

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void widen_vector(Raw<T, N>& raw, const Place& place, int half,
                                             int extent, float (&out)[N]) {
    if constexpr (!kWhole) {
        settle<Access::kLanes>(raw, place.column[half], extent);
    }
    widen<T, N>(raw, out);
}

// Each value rounded once to T, to nearest even, two with one instruction.
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> narrow_pairs(const float (&values)[N]) {
    if constexpr (sizeof(T) == 4) {
        return narrow<T, N>(values);
    } else {
        typedef float Two __attribute__((ext_vector_type(2)));
        typedef T Narrow __attribute__((ext_vector_type(2)));
        Raw<T, N> raw;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const Two two = {values[2 * i], values[2 * i + 1]};
            raw.words[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, Narrow));
        }
        return raw;
    }
}

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void store_vector(T* head, const Place& place, int half,
                                             const float (&values)[N]) {
    T* run = head + place.base[half];
    if constexpr (kWhole) {
        if (place.column[half] < place.extent) {
            const Raw<T, N> raw = narrow_pairs<T, N>(values);
            constexpr int kWords = Raw<T, N>::kWords;
            using W = WordVector<kWords, static_cast<int>(sizeof(T))>;
            typename W::plain words;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                words[i] = raw.words[i];
            }
            __builtin_nontemporal_store(
                words, reinterpret_cast<typename W::type*>(run + place.column[half]));
        }
    } else {
        store<Access::kLanes, kForwardStores, T, N>(run, place.column[half], place.extent,
                                                    narrow_pairs<T, N>(values));
    }
}

// A lane's part of a norm's weight; zeros where it has no columns.
template <bool kWhole, typename W, int N>
__device__ __forceinline__ void load_weight(const void* weight, const Place& place,
                                            float (&out)[2][N]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const W* run = static_cast<const W*>(weight) + place.base[half];
        Raw<W, N> raw{};
        if constexpr (kWhole) {
            if (place.column[half] < place.extent) {
                __builtin_memcpy(&raw, run + place.column[half], sizeof(raw));
            }
        } else {
            raw = load<Access::kLanes, W, N, kCached>(run, place.column[half], place.extent);
            settle<Access::kLanes>(raw, place.column[half], place.extent);
        }
        widen<W, N>(raw, out[half]);
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
        const float turned = __builtin_fmaf(x, c, -(y * s));
        y = __builtin_fmaf(x, s, y * c);
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

// Sum over each aligned run of `lanes` lanes, a power of two; kLanes: the number where
// it is known at compile time, else 0.
template <int kLanes>
__device__ __forceinline__ float head_sum(float value, int lanes) {
    const int own = kLanes > 0 ? kLanes : lanes;
#define ROTARY_ADD(control) \
    value += __builtin_bit_cast(float, RMS_DPP(__builtin_bit_cast(uint32_t, value), control))
    if (own > 1) {
        ROTARY_ADD(kXor1);
    }
    if (own > 2) {
        ROTARY_ADD(kXor2);
    }
    if (own > 4) {
        ROTARY_ADD(kHalfMirror);
    }
    if (own > 8) {
        ROTARY_ADD(kMirror);
    }
#undef ROTARY_ADD
    if (own > 16) {
        value += __shfl_xor(value, 16);
    }
    if (own > 32) {
        value += __shfl_xor(value, 32);
    }
    return value;
}

// 1 / sqrt(value), within two units in the last place: the hardware's reciprocal root
// (one unit) where it takes the value whole, the exact operations under that.
__device__ __forceinline__ float inverse_root(float value) {
    return value >= 0x1p-120f ? __builtin_amdgcn_rsqf(value) : 1.0f / __builtin_sqrtf(value);
}

// ----------------------------------------------------------------------------
// One block per item, a tile of tokens and a share of their heads on one side; in the
// backward with a norm the blocks walk the items, so that each leaves one row of
// partial sums, which reduce_kernel adds in a fixed order.

// What a lane reads of a head: what is turned, and the backward's heads.
template <typename T, int N, bool kSums>
struct Head {
    Raw<T, N> turned[2];
    Raw<T, N> heads[kSums ? 2 : 1];
    int local;  // its token in the tile
};

// Waves for each SIMD. The backward of eight pairs a lane needs 140 registers: held to
// 128 it left 23 of them for memory, and wrote and read more there than its tensors have
// ([8192, 24 heads of 64] fp16 41 against 33 us).
constexpr int waves_of(Pass pass, int columns) {
    if (pass == Pass::kTurn) {
        return columns == 8 ? 5 : 6;
    }
    return columns == 8 ? (pass == Pass::kNormBackward ? 3 : 4)
                        : pass == Pass::kNormBackward ? 4 : 5;
}

template <typename T, int N, Pass kPass, bool kWhole, int kLanes>
__global__ __launch_bounds__(kThreads, waves_of(kPass, N)) void heads_kernel(Args a) {
    constexpr bool kNormed = kPass != Pass::kTurn;
    constexpr bool kSums = kPass == Pass::kNormBackward;
    // Without a norm there is little to do while the next head comes, and more waves
    // fit instead ([3711, 20 heads of 80] fp32 11.7 against 12.9 us).
    constexpr bool kAhead = kPass != Pass::kTurn;
    // Cosines and sines [tile][row_pairs] each; at the end the sums.
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int which = static_cast<int>(blockIdx.x) < a.side[0].blocks ? 0 : 1;
    const Side& side = a.side[which];
    const int block = static_cast<int>(blockIdx.x) - (which == 0 ? 0 : a.side[0].blocks);
    float* cosines = lds;
    float* sines = lds + side.tile * a.row_pairs;
    const int lanes = kLanes > 0 ? kLanes : a.lanes;
    const int shift = kLanes > 0 ? __builtin_ctz(kLanes > 0 ? kLanes : 1) : a.lanes_shift;
    const int chunk = static_cast<int>(threadIdx.x) & (lanes - 1);
    const int slot = static_cast<int>(threadIdx.x) >> shift;
    const int slots = kThreads >> shift;
    const Place place = place_of<N>(a, chunk);
    const bool turns = place.pair >= 0;
    const bool normed = kNormed && side.weight != nullptr;
    const bool one_run = a.inner >= a.tokens;
    // A lane's head: its token in the tile, and where it is.
    int local = 0;
    int head = 0;
    const T* heads = nullptr;
    const T* grad = nullptr;
    const auto find_head = [&](int begin, int row) {
        local = static_cast<int>((static_cast<float>(row) + 0.5f) * side.inverse_count);
        head = row - local * side.count;
        int outer = 0;
        int within = begin + local;
        if (!one_run) {
            outer = within / a.inner;
            within -= outer * a.inner;
        }
        heads = static_cast<const T*>(side.heads) + outer * side.heads_outer
            + within * side.heads_token + head * side.heads_head;
        if constexpr (kSums) {
            grad = static_cast<const T*>(side.grad) + outer * side.grad_outer
                + within * side.grad_token + head * side.grad_head;
        }
    };
    const auto next_head = [&](int begin, int row) {
        if (!one_run) {
            find_head(begin, row);
            return;
        }
        local += side.step_tokens;
        head += side.step_heads;
        const bool wraps = head >= side.count;
        local += wraps ? 1 : 0;
        head -= wraps ? side.count : 0;
        heads += side.heads_step + (wraps ? side.heads_wrap : 0);
        if constexpr (kSums) {
            grad += side.grad_step + (wraps ? side.grad_wrap : 0);
        }
    };
    const auto load_head = [&](Head<T, N, kSums>* out) {
        const T* turned = kSums ? grad : heads;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            out->turned[half] = load_vector<kWhole, T, N>(turned, place, half, place.extent);
            if constexpr (kSums) {
                out->heads[half] =
                    load_vector<kWhole, T, N>(heads, place, half, normed ? place.extent : 0);
            }
        }
        out->local = local;
    };
    float weight[2][N];
    float sums[2][N];
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        (&sums[0][0])[i] = 0.0f;
        (&weight[0][0])[i] = 1.0f;
    }
    Head<T, N, kSums> ahead;
    for (int item = block; item < side.items; item += side.blocks) {
        const int tile = side.parts == 1 ? item : item / side.parts;
        const int first_row = slot + (item - tile * side.parts) * slots;
        const int begin = tile * side.tile;
        const int tokens = a.tokens - begin < side.tile ? a.tokens - begin : side.tile;
        const int rows = tokens * side.count;
        // A tile's first heads are read while its angles are made.
        if (first_row < rows) {
            find_head(begin, first_row);
            load_head(&ahead);
        }
        if (normed && item == block) {
            if (side.weight_dtype == RLN_DTYPE_F32) {
                load_weight<kWhole, float, N>(side.weight, place, weight);
            } else if (side.weight_dtype == RLN_DTYPE_F16) {
                load_weight<kWhole, half_t, N>(side.weight, place, weight);
            } else {
                load_weight<kWhole, bf16_t, N>(side.weight, place, weight);
            }
        }
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
        for (int row = first_row; row < rows; row += side.row_step) {
            if (!kAhead && row > first_row) {
                next_head(begin, row);
                load_head(&ahead);
            }
            Head<T, N, kSums> now = ahead;
            if (kAhead && row + side.row_step < rows) {
                next_head(begin, row + side.row_step);
                load_head(&ahead);
            }
            const int angle = now.local * a.row_pairs + (turns ? place.pair : 0);
            float values[2][N];
            float cosine[N];
            float sine[N];
            read_lds<N>(cosines + angle, cosine);
            read_lds<N>(sines + angle, sine);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                widen_vector<kWhole, T, N>(now.turned[half], place, half, place.extent,
                                           values[half]);
            }
            if constexpr (kPass == Pass::kNorm) {
                if (normed) {
                    float sum = 0.0f;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            sum = __builtin_fmaf(values[half][e], values[half][e], sum);
                        }
                    }
                    sum = head_sum<kLanes>(sum, lanes);
                    const float rstd =
                        inverse_root(sum * a.inverse_size + a.eps);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            values[half][e] *= rstd * weight[half][e];
                        }
                    }
                }
            }
            // Not by a cosine of 1 and a sine of 0: each of the other values stays, also
            // beside one that is not finite.
            if (turns) {
                turn<N>(values[0], values[1], cosine, sine, a.interleaved != 0);
            }
            if constexpr (kSums) {
                if (normed) {
                    float unit[2][N];
                    float square = 0.0f;
                    float shared = 0.0f;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        widen_vector<kWhole, T, N>(now.heads[half], place, half, place.extent,
                                                   unit[half]);
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            square = __builtin_fmaf(unit[half][e], unit[half][e], square);
                            shared = __builtin_fmaf(values[half][e] * weight[half][e],
                                                    unit[half][e], shared);
                        }
                    }
                    square = head_sum<kLanes>(square, lanes);
                    shared = head_sum<kLanes>(shared, lanes);
                    const float rstd =
                        inverse_root(square * a.inverse_size + a.eps);
                    shared *= rstd * a.inverse_size;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            const float normal = unit[half][e] * rstd;
                            sums[half][e] =
                                __builtin_fmaf(values[half][e], normal, sums[half][e]);
                            values[half][e] = rstd
                                * __builtin_fmaf(-normal, shared,
                                                 values[half][e] * weight[half][e]);
                        }
                    }
                }
            }
            T* to = static_cast<T*>(side.output)
                + (static_cast<int64_t>(begin) * side.count + row) * a.size;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                store_vector<kWhole, T, N>(to, place, half, values[half]);
            }
        }
        __syncthreads();  // the tile's angles are read before the next one's are written
    }
    if constexpr (kSums) {
        if (side.partials == nullptr) {
            return;
        }
        // The wave's heads by exchanges, the block's waves through LDS, in their order.
        constexpr int kWaves = kThreads / kWave;
        const int wave = static_cast<int>(threadIdx.x) / kWave;
        const int lane = static_cast<int>(threadIdx.x) % kWave;
        const int vectors = 2 * a.lanes;  // [lanes][2] of N
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float sum = sums[half][e];
                for (int other = a.lanes; other < kWave; other *= 2) {
                    sum += __shfl_xor(sum, other);
                }
                if (lane < a.lanes) {
                    lds[(wave * vectors + chunk * 2 + half) * N + e] = sum;
                }
            }
        }
        __syncthreads();
        float* partial = side.partials + static_cast<int64_t>(block) * a.size;
        for (int i = static_cast<int>(threadIdx.x); i < vectors * N; i += kThreads) {
            const int e = i % N;
            const int half = i / N & 1;
            const Place at = place_of<N>(a, i / N >> 1);
            if (at.column[half] + e < at.extent) {
                float sum = lds[i];
#pragma unroll
                for (int other = 1; other < kWaves; ++other) {
                    sum += lds[other * vectors * N + i];
                }
                partial[at.base[half] + at.column[half] + e] = sum;
            }
        }
    }
}

// Fixed-order sums of the partials [blocks][size], rounded once to the weights'
// types. A block owns 16 columns of one side; its 64 groups of 16 lanes take every 64th
// row, all reads of eight rows and of the groups' totals under way together.
constexpr int kReduceColumns = 16;
constexpr int kReduceGroups = 64;

struct ReduceArgs {
    const float* partials[2];
    void* grad_weight[2];
    int dtype[2];
    int blocks[2];
    int size;
};

__global__ __launch_bounds__(kReduceColumns * kReduceGroups) void reduce_kernel(ReduceArgs a) {
    __shared__ float totals[kReduceGroups][kReduceColumns];
    const int which = blockIdx.y;
    if (a.grad_weight[which] == nullptr) {
        return;
    }
    const int lane = threadIdx.x % kReduceColumns;
    const int group = threadIdx.x / kReduceColumns;
    const int column = blockIdx.x * kReduceColumns + lane;
    float total = 0.0f;
    if (column < a.size) {
        constexpr int kBatch = 8;
        const int blocks = a.blocks[which];
        const float* from = a.partials[which] + static_cast<int64_t>(group) * a.size + column;
        const int64_t step = static_cast<int64_t>(kReduceGroups) * a.size;
        for (int block = group; block < blocks; block += kBatch * kReduceGroups) {
            float values[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                values[i] = block + i * kReduceGroups < blocks ? from[i * step] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                total += values[i];
            }
            from += kBatch * step;
        }
    }
    totals[group][lane] = total;
    __syncthreads();
    if (group == 0 && column < a.size) {
        float sum = 0.0f;
#pragma unroll
        for (int other = 0; other < kReduceGroups; ++other) {
            sum += totals[other][lane];
        }
        store_one(a.grad_weight[which], a.dtype[which], column, sum);
    }
}

// ----------------------------------------------------------------------------
// Launch shapes and checks (host).

struct Grid {
    int columns;   // of a lane's vector
    int lanes;
    int lanes_shift;
    int turned_lanes;
    int row_pairs;
    bool whole;
    struct {
        int tile;
        int parts;
        int items;
        int blocks;
    } side[2];
};

// Tiles: the blocks that a CU holds at once make `resident` of the launch; each costs
// its passes, the turns of its lanes over the tile's heads, and half of one more for its
// start and its angles, one and a half in a forward with a norm. The tiles (powers of two,
// both sides with about the same passes) are those of the least time by that count,
// rounds of blocks times a block's cost ([16384, 32 + 8 heads of 128] bf16 69 us in tiles
// of 4 passes, 79 of 8, 89 of 2; [8858, 16 + 16 of 72] fp16 29 of 4, 23 of 16). Where even
// tiles of one token are too few blocks, several share a tile's heads. A backward with
// sums walks its items with the resident blocks.
Grid grid_of(int64_t tokens, const int64_t (&counts)[2], int64_t size, int64_t pairs, int dtype,
             Pass pass) {
    Grid grid{};
    const int left = static_cast<int>(size - 2 * pairs);
    const auto whole = [&](int columns) {
        return pairs % columns == 0 && left % (2 * columns) == 0;
    };
    grid.columns = columns_of(dtype);
    if (!whole(grid.columns) && whole(4)) {
        grid.columns = 4;
    }
    const int columns = grid.columns;
    grid.whole = whole(columns);
    grid.turned_lanes = static_cast<int>((pairs + columns - 1) / columns);
    const int vectors = grid.turned_lanes + (left + 2 * columns - 1) / (2 * columns);
    grid.lanes = 1;
    while (grid.lanes < vectors) {
        grid.lanes *= 2;
        ++grid.lanes_shift;
    }
    grid.row_pairs = grid.turned_lanes * columns;
    const int64_t slots = kThreads / grid.lanes;
    const int64_t resident = waves_of(pass, columns) * kComputeUnits;
    const auto divided = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    int64_t least = INT64_MAX;
    for (int64_t goal = 1; goal <= 32; goal *= 2) {
        int64_t tile[2] = {0, 0};
        int64_t blocks = 0;
        int64_t passes = 0;
        for (int i = 0; i < 2; ++i) {
            if (counts[i] > 0) {
                tile[i] = 1;
                while (tile[i] * counts[i] < goal * slots
                       && 2 * tile[i] * grid.row_pairs <= kTilePairs) {
                    tile[i] *= 2;
                }
                blocks += divided(tokens, tile[i]);
                const int64_t own = divided(tile[i] * counts[i], slots);
                passes = own > passes ? own : passes;
            }
        }
        const int64_t start = pass == Pass::kNorm ? 3 : 1;
        const int64_t cost = divided(blocks, resident) * (start + 2 * passes);
        if (cost < least) {
            least = cost;
            grid.side[0].tile = static_cast<int>(tile[0]);
            grid.side[1].tile = static_cast<int>(tile[1]);
        }
    }
    for (int i = 0; i < 2; ++i) {
        if (counts[i] == 0) {
            continue;
        }
        auto& side = grid.side[i];
        const int64_t share = resident * counts[i] / (counts[0] + counts[1]);
        const int64_t tiles = divided(tokens, side.tile);
        const int64_t passes = divided(side.tile * counts[i], slots);
        const int64_t parts = share / tiles > 1 ? share / tiles : 1;
        side.parts = static_cast<int>(passes < parts ? passes : parts);
        side.items = static_cast<int>(tiles * side.parts);
        // A launch holds fewer than 2^32 threads.
        int64_t most = int64_t{1} << 22;
        if (pass == Pass::kNormBackward) {
            most = share > 0 ? share : 1;
        }
        side.blocks = static_cast<int>(side.items < most ? side.items : most);
    }
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
    // The rows of a tile are divided by the count in fp32.
    if (given->count < 0 || given->count > kMaxHeads) {
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
    if (given->pairs < 1 || given->pairs > size / 2) {
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
    const int64_t counts[2] = {a->side[0].count, a->side[1].count};
    if (counts[0] == 0 && counts[1] == 0) {
        return fail(RLN_ERR_INVALID, "empty tensors are unsupported");
    }
    if ((status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    *normed = a->side[0].weight != nullptr || a->side[1].weight != nullptr;
    if (backward && !*normed) {
        for (Side& side : a->side) {
            side.heads = side.grad;
            side.heads_outer = side.grad_outer;
            side.heads_token = side.grad_token;
            side.heads_head = side.grad_head;
        }
    }
    *grid = grid_of(outer * inner, counts, size, a->pairs, dtype,
                    !*normed ? Pass::kTurn : backward ? Pass::kNormBackward : Pass::kNorm);
    for (int i = 0; i < 2; ++i) {
        a->side[i].tile = grid->side[i].tile;
        a->side[i].parts = grid->side[i].parts;
        a->side[i].items = grid->side[i].items;
        a->side[i].blocks = grid->side[i].blocks;
        Side& side = a->side[i];
        if (side.count > 0) {
            side.row_step = kThreads / grid->lanes * side.parts;
            side.step_tokens = side.row_step / side.count;
            side.step_heads = side.row_step % side.count;
            // Unsigned: a step past the last token may not fit, and is not taken.
            const auto step = [&](int64_t token, int64_t head) {
                return static_cast<int64_t>(
                    static_cast<uint64_t>(side.step_tokens) * static_cast<uint64_t>(token)
                    + static_cast<uint64_t>(side.step_heads) * static_cast<uint64_t>(head));
            };
            side.heads_step = step(side.heads_token, side.heads_head);
            side.heads_wrap = side.heads_token - side.count * side.heads_head;
            side.grad_step = step(side.grad_token, side.grad_head);
            side.grad_wrap = side.grad_token - side.count * side.grad_head;
        }
    }
    a->tokens = static_cast<int>(outer * inner);
    a->inner = static_cast<int>(inner);
    a->size = static_cast<int>(size);
    a->row_pairs = grid->row_pairs;
    a->inverse_row_pairs = 1.0f / static_cast<float>(grid->row_pairs);
    a->lanes = grid->lanes;
    a->lanes_shift = grid->lanes_shift;
    a->turned_lanes = grid->turned_lanes;
    a->backward = backward;
    a->eps = static_cast<float>(eps);
    a->inverse_size = 1.0f / static_cast<float>(size);
    return RLN_OK;
}

template <typename T, int N, Pass kPass>
int launch(const Args& a, const Grid& grid, hipStream_t stream) {
    const int tile = a.side[0].tile > a.side[1].tile ? a.side[0].tile : a.side[1].tile;
    size_t floats = 2 * static_cast<size_t>(tile) * a.row_pairs;
    const size_t sums = static_cast<size_t>(kThreads / kWave) * 2 * a.lanes * N;
    if (kPass == Pass::kNormBackward && floats < sums) {
        floats = sums;  // in the place of the angles
    }
    // Sums over the lanes of the usual head sizes without a choice at run time.
    auto kernel =
        grid.whole ? heads_kernel<T, N, kPass, true, 0> : heads_kernel<T, N, kPass, false, 0>;
    if constexpr (kPass != Pass::kTurn) {
        if (grid.whole) {
            kernel = a.lanes == 4 ? heads_kernel<T, N, kPass, true, 4>
                : a.lanes == 8    ? heads_kernel<T, N, kPass, true, 8>
                : a.lanes == 16   ? heads_kernel<T, N, kPass, true, 16>
                                  : kernel;
        }
    }
    const unsigned blocks = static_cast<unsigned>(a.side[0].blocks + a.side[1].blocks);
    kernel<<<dim3(blocks), kThreads, floats * sizeof(float), stream>>>(a);
    return check_launch("rotary heads_kernel");
}

template <typename T, int N>
int launch_pass(const Args& a, const Grid& grid, bool normed, hipStream_t stream) {
    if (!normed) {
        return launch<T, N, Pass::kTurn>(a, grid, stream);
    }
    return a.backward ? launch<T, N, Pass::kNormBackward>(a, grid, stream)
                      : launch<T, N, Pass::kNorm>(a, grid, stream);
}

template <typename T>
int launch_columns(const Args& a, const Grid& grid, bool normed, hipStream_t stream) {
    if (grid.columns == kColumns<T>) {
        return launch_pass<T, kColumns<T>>(a, grid, normed, stream);
    }
    return launch_pass<T, 4>(a, grid, normed, stream);
}

int launch_dtype(const Args& a, const Grid& grid, int dtype, bool normed, void* stream) {
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case RLN_DTYPE_F32:
            return launch_columns<float>(a, grid, normed, queue);
        case RLN_DTYPE_F16:
            return launch_columns<half_t>(a, grid, normed, queue);
        default:
            return launch_columns<bf16_t>(a, grid, normed, queue);
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
    if (!float_dtype(dtype) || outer < 1 || inner < 1 || inner > INT32_MAX / 2
        || outer > INT32_MAX / 2 / inner || size < 1 || size > kMaxSize || pairs < 1
        || pairs > size / 2 || q_heads < 0 || k_heads < 0 || q_heads > kMaxHeads
        || k_heads > kMaxHeads) {
        return 0;
    }
    const int64_t counts[2] = {q_heads, k_heads};
    const Grid grid = grid_of(outer * inner, counts, size, pairs, dtype, Pass::kNormBackward);
    return (static_cast<size_t>(grid.side[0].blocks) + grid.side[1].blocks)
        * static_cast<size_t>(size) * sizeof(float);
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
            (static_cast<size_t>(a.side[0].blocks) + a.side[1].blocks)
            * static_cast<size_t>(size) * sizeof(float);
        if (workspace == nullptr || workspace_bytes < needed) {
            return fail(RLN_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", needed,
                        workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
        }
        if ((status = check_address("workspace", workspace, 4)) != RLN_OK) {
            return status;
        }
        a.side[0].partials = static_cast<float*>(workspace);
        a.side[1].partials =
            a.side[0].partials + static_cast<int64_t>(a.side[0].blocks) * a.size;
    }
    status = launch_dtype(a, grid, dtype, normed, stream);
    if (status != RLN_OK || !sums) {
        return status;
    }
    for (int i = 0; i < 2; ++i) {
        reduce.partials[i] = a.side[i].partials;
        reduce.dtype[i] = a.side[i].weight_dtype;
        reduce.blocks[i] = a.side[i].blocks;
    }
    reduce.size = a.size;
    const unsigned blocks = static_cast<unsigned>((size + kReduceColumns - 1) / kReduceColumns);
    reduce_kernel<<<dim3(blocks, 2), kReduceColumns * kReduceGroups, 0,
                    static_cast<hipStream_t>(stream)>>>(reduce);
    return check_launch("rotary reduce_kernel");
}

}  // extern "C"
