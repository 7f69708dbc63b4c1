// Kernels of the root-mean-square norm with the residual's addition, its 8-bit
// output and its 8-bit checkpoint (include/rln.h, the rln_rms_* entry points).
//
// Per row of H values (u the new residual stream, rounded to x's type):
//
//   u = x + branch                      r = 1 / sqrt(sum(u^2) / H + eps)
//   normalized = (u * r) * weight
//   backward: p = gy * weight, c = sum(p * u * r) / H,
//             g = gu + r * (p - u * r * c),   grad_weight = sum_rows gy * u * r
//
// 8-bit outputs take steps of v = u * weight against the largest |v| of each
// group of columns. Since r is one positive factor of the whole row, it goes
// into the scale alone: code = round(v * (Q / max|v|)), scale = max|v| / Q * r.
// The codes therefore depend on no sum (they are the same for every split of a
// row over lanes), and the maximum and the sum of squares are taken in the same
// pass over the row. The 8-bit checkpoint of u does the same with u itself.
//
// Every pass is bound by memory (under 20 fp32 operations per element against
// 5-20 bytes), so a row is read once into registers, reduced there, and written
// from there. A row belongs to `parts` waves; vector j of the row (8 columns of
// a 16-bit stream, 4 of a 32-bit one: 16 bytes of the stream per lane) sits in
// slot v of lane l of part p with j = (v * parts + p) * 64 + l. `parts` is a
// run-time value, so any row length gets a team without idle waves. Short rows, of
// at most half a wave's vectors, take 8, 16 or 32 lanes each instead (Access::kLanes).
//
// A row is read and written in vectors, through one buffer descriptor per row and
// tensor where its rows start and end on whole 32-bit words (Access::kWords; 32-bit
// elements always do): words past the end of the row are dropped by the
// hardware's range check, without a branch, and stores carry a cache policy.
// 16- and 8-bit rows of other lengths, strides and alignments (Access::kElements)
// take global accesses, which the hardware serves in 128 bits at element
// alignment; the one vector that crosses the end of a row is read shifted and
// stored by elements.
#ifndef RMS_DEVICE_H
#define RMS_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rln.h"

namespace rln {

// Defined in rln_api.hip.
int fail(int code, const char* format, ...);
int check_launch(const char* what);
int check_stream(void* stream);
void clear_error();

namespace rms {

using half_t = _Float16;
using bf16_t = __bf16;
// Tag of a forward without a branch (the first norm of a stack): u = x, which
// is not written again.
struct NoBranch {};

constexpr int kWave = 64;
constexpr int64_t kMaxHidden = 16384;
constexpr int kMaxParts = 16;
constexpr int kCheckpointGroup = 128;
// As the shift of a column to its group: every column is in group 0.
constexpr int kWholeRow = 31;
// The least maximum of a group: keeps Q / max finite where a group is all
// zeros (or below 2^-100, far under any value a norm is fed).
constexpr float kLeastMaximum = 0x1p-100f;

// 16 bytes of the stream per lane and slot.
template <typename X>
constexpr int kColumns = 16 / static_cast<int>(sizeof(X));

// How rows are accessed (see above); kLanes: as kElements, for waves whose lanes
// hold several rows, where the others ask for one row per wave.
enum class Access { kWords, kElements, kLanes };

template <Access kAccess, typename T>
constexpr bool kBuffer =
    kAccess == Access::kWords || (kAccess == Access::kElements && sizeof(T) == 4);

enum class Mode { kNormalize, kCheckpoint, kQuantize };

struct ForwardArgs {
    const void* x;
    const void* branch;
    const void* weight;
    void* updated;
    void* normalized;   // or the codes
    float* rstd;        // may be null
    int8_t* checkpoint;
    float* scale;       // of the checkpoint or of the codes
    int64_t x_stride;
    int64_t branch_stride;
    int64_t rows;
    int hidden;
    int parts;
    int row_lanes;      // of Access::kLanes
    int words;          // Access::kWords serves every tensor
    int weight_dtype;
    int output_dtype;   // normalized's, or the codes'
    int group_shift;    // log2 of the columns under one scale, or kWholeRow
    int groups;         // scales per row
    float eps;
    float inv_hidden;
};

struct BackwardArgs {
    const void* grad_updated;  // may be null
    const void* grad_normalized;
    const void* updated;
    const int8_t* checkpoint;
    const float* scale;
    const void* weight;
    const float* rstd;
    void* grad_x;
    void* grad_branch;  // null where it equals grad_x
    float* partials;    // [blocks][hidden] of a walk, or null
    void* grad_weight;  // of a launch with slab blocks
    int slabs;          // its first blocks
    int64_t updated_stride;
    int64_t rows;
    int hidden;
    int parts;
    int row_lanes;
    int words;
    int groups;
    int weight_dtype;
    int branch_dtype;
    float inv_hidden;
};

// ----------------------------------------------------------------------------
// Vectors of N elements as raw words, at element alignment.

template <int Words, int Alignment>
struct WordVector;
#define RMS_WORDS(count, alignment)                                                     \
    template <>                                                                         \
    struct WordVector<count, alignment> {                                                   \
        typedef uint32_t plain __attribute__((ext_vector_type(count)));                 \
        typedef plain type __attribute__((aligned(alignment)));                         \
    }
RMS_WORDS(4, 4);
RMS_WORDS(4, 2);
RMS_WORDS(2, 4);
RMS_WORDS(2, 2);
RMS_WORDS(2, 1);
#undef RMS_WORDS
#define RMS_WORD(alignment)                                                             \
    template <>                                                                         \
    struct WordVector<1, alignment> {                                                   \
        typedef uint32_t plain;                                                         \
        typedef uint32_t type __attribute__((aligned(alignment)));                      \
    }
RMS_WORD(4);
RMS_WORD(2);
RMS_WORD(1);
#undef RMS_WORD
typedef uint16_t AnyHalf __attribute__((aligned(1)));

// N elements of T as 32-bit words.
template <typename T, int N>
struct Raw {
    static constexpr int kWords = N * static_cast<int>(sizeof(T)) / 4;
    uint32_t words[kWords];
};

// Cache policies of buffer accesses: bit 0 is sc0, bit 1 nt, bit 4 sc1.
// Rows pass once and are read non-temporally; the weight stays cached. Forward
// outputs are stored non-temporally, the backward's and the widening's written
// through: measured against plain stores, [16384, 4096] bf16 forward 84.0 against
// 90.3 us (write-through 85.5), [6001, 2880] 25.6 against 28.2 (26.3), [8192, 8192]
// fp32 backward with the checkpoint 157.0 against 170.4 (non-temporal 159.8),
// [16384, 2048] bf16 44.2 against 46.1 (45.6). All over buffers that pass the caches;
// what a small launch's consumer pays for outputs it might have found there was not
// measured.
constexpr int kCached = 0;
constexpr int kOnce = 2;
constexpr int kForwardStores = 2;
constexpr int kBackwardStores = 17;

// A descriptor over `count` elements at a wave-uniform address, whole words
// (count 0: nothing is read or written through it, wherever it points). Accesses
// of several words are range-checked word by word.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* row, int count) {
    const uint64_t bits = reinterpret_cast<uint64_t>(row);
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits));
    const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void*>(static_cast<uint64_t>(high) << 32 | low), 0,
        __builtin_amdgcn_readfirstlane(count * static_cast<int>(sizeof(T))), 0x00020000);
}

// Elements [column, column + N) of a row of `hidden` (both wave-uniform but for
// the column), zeros past its end; settle() has to follow before they are used.
template <Access kAccess, typename T, int N, int Policy = kOnce>
__device__ __forceinline__ Raw<T, N> load(const T* __restrict__ row, int column, int hidden) {
    Raw<T, N> raw;
    constexpr int kWords = Raw<T, N>::kWords;
    constexpr int kChunk = kWords < 4 ? kWords : 4;
    if constexpr (kBuffer<kAccess, T>) {
        const auto buffer = row_buffer(row, hidden);
#pragma unroll
        for (int i = 0; i < kWords; i += kChunk) {
            const int offset = column * static_cast<int>(sizeof(T)) + 4 * i;
            if constexpr (kChunk == 4) {
                const auto words = __builtin_amdgcn_raw_buffer_load_b128(buffer, offset, 0, Policy);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    raw.words[i + k] = words[k];
                }
            } else if constexpr (kChunk == 2) {
                const auto words = __builtin_amdgcn_raw_buffer_load_b64(buffer, offset, 0, Policy);
                raw.words[i] = words[0];
                raw.words[i + 1] = words[1];
            } else {
                raw.words[i] = __builtin_amdgcn_raw_buffer_load_b32(buffer, offset, 0, Policy);
            }
        }
        return raw;
    }
    // Vectors of up to 16 bytes; one that crosses the row's end is read from the
    // row's last whole vector, so that no lane branches around memory, and shifted
    // down by settle(), so that no load waits for another.
    constexpr int kElements = 4 * kChunk / static_cast<int>(sizeof(T));
    using W = WordVector<kChunk, static_cast<int>(sizeof(T))>;
#pragma unroll
    for (int i = 0; i < kWords; i += kChunk) {
        const int begin = column + i / kChunk * kElements;
        typename W::plain words{};
        if (hidden >= kElements) {
            const int start = begin < hidden - kElements ? begin : hidden - kElements;
            const typename W::type* from = reinterpret_cast<const typename W::type*>(row + start);
            if constexpr (Policy == kOnce) {
                words = __builtin_nontemporal_load(from);
            } else {
                words = *from;
            }
        }
        if constexpr (kChunk == 1) {
            raw.words[i] = words;
        } else {
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                raw.words[i + k] = words[k];
            }
        }
    }
    if (hidden < kElements) {  // rows shorter than a vector, and no row at all
#pragma unroll
        for (int e = 0; e < kElements - 1; ++e) {
            if (column + e < hidden) {
                uint32_t element;
                if constexpr (sizeof(T) == 4) {
                    element = reinterpret_cast<const uint32_t*>(row)[column + e];
                } else if constexpr (sizeof(T) == 2) {
                    element = reinterpret_cast<const uint16_t*>(row)[column + e];
                } else {
                    element = reinterpret_cast<const uint8_t*>(row)[column + e];
                }
                constexpr int kPerWord = 4 / static_cast<int>(sizeof(T));
                raw.words[e / kPerWord] |=
                    element << (e % kPerWord * 8 * static_cast<int>(sizeof(T)));
            }
        }
    }
    return raw;
}

// The second half of load(): moves the vectors that were read from an earlier
// column to their place, zeros behind them. By elements under branches, or
// shifted right after each load, the loads of a row waited for one another
// ([8192, 4095] bf16 backward 121 and 85 us).
template <Access kAccess, typename T, int N>
__device__ __forceinline__ void settle(Raw<T, N>& raw, int column, int hidden) {
    if constexpr (!kBuffer<kAccess, T>) {
        constexpr int kWords = Raw<T, N>::kWords;
        constexpr int kChunk = kWords < 4 ? kWords : 4;
        constexpr int kElements = 4 * kChunk / static_cast<int>(sizeof(T));
#pragma unroll
        for (int i = 0; i < kWords; i += kChunk) {
            const int begin = column + i / kChunk * kElements;
            if (hidden >= kElements && begin > hidden - kElements) {
                unsigned __int128 bits = 0;
#pragma unroll
                for (int k = kChunk - 1; k >= 0; --k) {
                    bits = bits << 32 | raw.words[i + k];
                }
                const int shift = (begin - hidden + kElements) * 8 * static_cast<int>(sizeof(T));
                bits = begin < hidden ? bits >> shift : 0;
#pragma unroll
                for (int k = 0; k < kChunk; ++k) {
                    raw.words[i + k] = static_cast<uint32_t>(bits >> (32 * k));
                }
            }
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void widen(const Raw<T, N>& raw, float (&out)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if constexpr (sizeof(T) == 4) {
            out[e] = __builtin_bit_cast(float, raw.words[e]);
        } else if constexpr (__is_same(T, bf16_t)) {
            const uint32_t word = raw.words[e / 2];
            out[e] = __builtin_bit_cast(float, e % 2 ? word & 0xffff0000u : word << 16);
        } else if constexpr (__is_same(T, half_t)) {
            const uint32_t word = raw.words[e / 2];
            out[e] = static_cast<float>(__builtin_bit_cast(
                half_t, static_cast<uint16_t>(e % 2 ? word >> 16 : word & 0xffffu)));
        } else {  // int8_t
            const uint32_t word = raw.words[e / 4];
            out[e] = static_cast<float>(static_cast<int8_t>(word >> (e % 4 * 8)));
        }
    }
}

// Each value rounded once to T, to nearest even.
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> narrow(const float (&values)[N]) {
    Raw<T, N> raw;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            raw.words[e] = __builtin_bit_cast(uint32_t, values[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const T low = static_cast<T>(values[e]);
            const T high = static_cast<T>(values[e + 1]);
            raw.words[e / 2] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, low))
                | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, high)) << 16;
        }
    }
    return raw;
}

template <Access kAccess, int Policy, typename T, int N>
__device__ __forceinline__ void store(T* __restrict__ row, int column, int hidden,
                                      const Raw<T, N>& raw) {
    constexpr int kWords = Raw<T, N>::kWords;
    constexpr int kChunk = kWords < 4 ? kWords : 4;
    if constexpr (kBuffer<kAccess, T>) {
        const auto buffer = row_buffer(row, hidden);
#pragma unroll
        for (int i = 0; i < kWords; i += kChunk) {
            const int offset = column * static_cast<int>(sizeof(T)) + 4 * i;
            if constexpr (kChunk == 4) {
                const typename WordVector<4, 4>::plain words = {raw.words[i], raw.words[i + 1],
                                                            raw.words[i + 2], raw.words[i + 3]};
                __builtin_amdgcn_raw_buffer_store_b128(words, buffer, offset, 0, Policy);
            } else if constexpr (kChunk == 2) {
                const typename WordVector<2, 4>::plain words = {raw.words[i], raw.words[i + 1]};
                __builtin_amdgcn_raw_buffer_store_b64(words, buffer, offset, 0, Policy);
            } else {
                __builtin_amdgcn_raw_buffer_store_b32(raw.words[i], buffer, offset, 0, Policy);
            }
        }
    } else if (column + N <= hidden) {
        using W = WordVector<kChunk, static_cast<int>(sizeof(T))>;
#pragma unroll
        for (int i = 0; i < kWords; i += kChunk) {
            typename W::plain words;
            if constexpr (kChunk == 1) {
                words = raw.words[i];
            } else {
#pragma unroll
                for (int k = 0; k < kChunk; ++k) {
                    words[k] = raw.words[i + k];
                }
            }
            __builtin_nontemporal_store(
                words, reinterpret_cast<typename W::type*>(row + column) + i / kChunk);
        }
    } else if (column >= hidden) {
        return;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < N - 1; ++e) {
            if (column + e < hidden) {
                reinterpret_cast<uint32_t*>(row)[column + e] = raw.words[e];
            }
        }
    } else {
        // The row's last elements, in at most three pieces of falling size.
        unsigned __int128 bits = 0;
#pragma unroll
        for (int k = kWords - 1; k >= 0; --k) {
            bits = bits << 32 | raw.words[k];
        }
        const int count = hidden - column;
        int place = column;
#pragma unroll
        for (int piece = N / 2; piece >= 1; piece /= 2) {
            if (count & piece) {
                const int bytes = piece * static_cast<int>(sizeof(T));
                if (bytes == 8) {
                    using W = WordVector<2, static_cast<int>(sizeof(T))>;
                    const typename W::plain words = {static_cast<uint32_t>(bits),
                                                     static_cast<uint32_t>(bits >> 32)};
                    *reinterpret_cast<typename W::type*>(row + place) = words;
                } else if (bytes == 4) {
                    *reinterpret_cast<typename WordVector<1, static_cast<int>(sizeof(T))>::type*>(
                        row + place) = static_cast<uint32_t>(bits);
                } else if (bytes == 2) {
                    *reinterpret_cast<AnyHalf*>(row + place) = static_cast<uint16_t>(bits);
                } else {
                    *reinterpret_cast<uint8_t*>(row + place) = static_cast<uint8_t>(bits);
                }
                bits >>= 8 * bytes;
                place += piece;
            }
        }
    }
}

// The weight and the outputs choose their type at run time: a wave-uniform
// branch, where a template parameter would multiply the instances by three.
template <Access kAccess, int N>
__device__ __forceinline__ void load_weight(const void* weight, int dtype, int column, int hidden,
                                            float (&out)[N]) {
    if (dtype == RLN_DTYPE_F32) {
        auto raw = load<kAccess, float, N, kCached>(static_cast<const float*>(weight), column,
                                                    hidden);
        settle<kAccess>(raw, column, hidden);
        widen<float, N>(raw, out);
    } else if (dtype == RLN_DTYPE_F16) {
        auto raw = load<kAccess, half_t, N, kCached>(static_cast<const half_t*>(weight), column,
                                                     hidden);
        settle<kAccess>(raw, column, hidden);
        widen<half_t, N>(raw, out);
    } else {
        auto raw = load<kAccess, bf16_t, N, kCached>(static_cast<const bf16_t*>(weight), column,
                                                     hidden);
        settle<kAccess>(raw, column, hidden);
        widen<bf16_t, N>(raw, out);
    }
}

template <Access kAccess, int Policy, int N>
__device__ __forceinline__ void store_as(void* tensor, int dtype, int64_t first, int column,
                                         int hidden, const float (&values)[N]) {
    if (dtype == RLN_DTYPE_F32) {
        store<kAccess, Policy, float, N>(static_cast<float*>(tensor) + first, column, hidden,
                                         narrow<float, N>(values));
    } else if (dtype == RLN_DTYPE_F16) {
        store<kAccess, Policy, half_t, N>(static_cast<half_t*>(tensor) + first, column, hidden,
                                          narrow<half_t, N>(values));
    } else {
        store<kAccess, Policy, bf16_t, N>(static_cast<bf16_t*>(tensor) + first, column, hidden,
                                          narrow<bf16_t, N>(values));
    }
}

// One value of a small tensor.
__device__ __forceinline__ void store_one(void* tensor, int dtype, int64_t index, float value) {
    if (dtype == RLN_DTYPE_F32) {
        static_cast<float*>(tensor)[index] = value;
    } else if (dtype == RLN_DTYPE_F16) {
        static_cast<half_t*>(tensor)[index] = static_cast<half_t>(value);
    } else {
        static_cast<bf16_t*>(tensor)[index] = static_cast<bf16_t>(value);
    }
}

// ----------------------------------------------------------------------------
// 8-bit codes.

// Round to nearest even, clipped to +-127.
template <int N>
__device__ __forceinline__ Raw<int8_t, N> narrow_int8(const float (&steps)[N]) {
    Raw<int8_t, N> raw;
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float whole = __builtin_rintf(steps[4 * w + e]);
            const int code =
                static_cast<int>(__builtin_fminf(__builtin_fmaxf(whole, -127.0f), 127.0f));
            word |= (static_cast<uint32_t>(code) & 0xffu) << (8 * e);
        }
        raw.words[w] = word;
    }
    return raw;
}

// e4m3 (OCP, the hardware's conversion rounds to nearest even), clipped to +-448.
template <int N>
__device__ __forceinline__ Raw<int8_t, N> narrow_e4m3(const float (&steps)[N]) {
    Raw<int8_t, N> raw;
    float clipped[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        clipped[e] = __builtin_fminf(__builtin_fmaxf(steps[e], -448.0f), 448.0f);
    }
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(clipped[4 * w], clipped[4 * w + 1], 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(clipped[4 * w + 2], clipped[4 * w + 3], word, true);
        raw.words[w] = static_cast<uint32_t>(word);
    }
    return raw;
}

template <int N>
__device__ __forceinline__ void widen_e4m3(const Raw<int8_t, N>& raw, float (&out)[N]) {
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        const int word = static_cast<int>(raw.words[w]);
        out[4 * w] = __builtin_amdgcn_cvt_f32_fp8(word, 0);
        out[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8(word, 1);
        out[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8(word, 2);
        out[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8(word, 3);
    }
}

// Bits of |value|: as unsigned integers they order like the magnitudes, with
// every NaN above infinity, so an integer maximum lets a NaN through (a
// floating one drops it).
__device__ __forceinline__ uint32_t magnitude_bits(float value) {
    return __builtin_bit_cast(uint32_t, value) & 0x7fffffffu;
}

struct GroupScale {
    float inverse;  // steps per unit
    float step;     // units per step
};

// Q / max and max / Q, each rounded once (correctly rounded divisions). A group
// that holds an infinity or a NaN gets NaN for its step: its values widen to NaN.
__device__ __forceinline__ GroupScale group_scale(uint32_t maximum_bits, float top) {
    const float maximum = __builtin_fmaxf(__builtin_bit_cast(float, maximum_bits), kLeastMaximum);
    GroupScale scale{top / maximum, maximum / top};
    if (maximum_bits >= 0x7f800000u) {
        scale = GroupScale{0.0f, __builtin_bit_cast(float, 0x7fc00000u)};
    }
    return scale;
}

// ----------------------------------------------------------------------------
// Reductions.

#define RMS_DPP(value, control) \
    __builtin_amdgcn_update_dpp(0, static_cast<int>(value), (control), 0xF, 0xF, false)
constexpr int kXor1 = 0xB1;         // quad_perm:[1,0,3,2]
constexpr int kXor2 = 0x4E;         // quad_perm:[2,3,0,1]
constexpr int kHalfMirror = 0x141;  // within 8 lanes
constexpr int kMirror = 0x140;      // within 16 lanes

// Sum over the wave's 64 lanes, the same value in every lane.
__device__ __forceinline__ float wave_sum(float value) {
#define RMS_ADD(control) \
    value += __builtin_bit_cast(float, RMS_DPP(__builtin_bit_cast(uint32_t, value), control))
    RMS_ADD(kXor1);
    RMS_ADD(kXor2);
    RMS_ADD(kHalfMirror);
    RMS_ADD(kMirror);
#undef RMS_ADD
    const int bits = __builtin_bit_cast(int, value);
    const float low = __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 0))
        + __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 16));
    const float high = __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 32))
        + __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 48));
    return low + high;
}

// Sum over each aligned run of `lanes` lanes (8, 16 or 32).
__device__ __forceinline__ float lanes_sum(float value, int lanes) {
#define RMS_ADD(control) \
    value += __builtin_bit_cast(float, RMS_DPP(__builtin_bit_cast(uint32_t, value), control))
    RMS_ADD(kXor1);
    RMS_ADD(kXor2);
    RMS_ADD(kHalfMirror);
    if (lanes > 8) {
        RMS_ADD(kMirror);
    }
#undef RMS_ADD
    return lanes > 16 ? value + __shfl_xor(value, 16) : value;
}

__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return a > b ? a : b;
}

// Maximum over each aligned run of `lanes` lanes (4, 8, 16, 32 or 64).
__device__ __forceinline__ uint32_t lanes_max(uint32_t value, int lanes) {
    value = larger(value, RMS_DPP(value, kXor1));
    value = larger(value, RMS_DPP(value, kXor2));
    if (lanes > 4) {
        value = larger(value, RMS_DPP(value, kHalfMirror));
    }
    if (lanes > 8) {
        value = larger(value, RMS_DPP(value, kMirror));
    }
    if (lanes > 16) {
        value = larger(value, __shfl_xor(value, 16));
    }
    if (lanes > 32) {
        value = larger(value, __shfl_xor(value, 32));
    }
    return value;
}

// The wave's index in its block and, from it, its row team and part.
struct Team {
    int wave;
    int index;  // row team in the block
    int part;
    int teams;
};

// A lane's place: its row among those its wave holds, and its lane of that row.
// A wave holds one row (or a part of one), or 64 / row_lanes short ones (kLanes).
struct Place {
    int rows;
    int row;
    int lane;
};

template <Access kAccess>
__device__ __forceinline__ Place place_of(int row_lanes) {
    const int lane = threadIdx.x % kWave;
    if constexpr (kAccess == Access::kLanes) {
        const int row = lane / row_lanes;
        return Place{kWave / row_lanes, row, lane - row * row_lanes};
    } else {
        return Place{1, 0, lane};
    }
}

__device__ __forceinline__ Team team_of(int parts) {
    Team team;
    team.wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    team.index = team.wave / parts;
    team.part = team.wave - team.index * parts;
    team.teams = static_cast<int>(blockDim.x) / (kWave * parts);
    return team;
}

// ----------------------------------------------------------------------------
// Forward: one row per team and turn. The grid covers the rows up to
// kMaxBlocks (a launch holds fewer than 2^32 threads); past that the
// teams walk.

template <typename X, typename B, int V, Mode kMode, Access kAccess>
__global__ __launch_bounds__(kMaxParts * kWave) void forward_kernel(ForwardArgs a) {
    constexpr int N = kColumns<X>;
    constexpr bool kBranch = !__is_same(B, NoBranch);
    __shared__ float sums[2][kMaxParts];
    __shared__ uint32_t maxima[2][kMaxParts];
    const Team team = team_of(a.parts);
    const Place place = place_of<kAccess>(a.row_lanes);
    const int block_rows = team.teams * place.rows;
    const int64_t step = static_cast<int64_t>(gridDim.x) * block_rows;
    int turn = 0;
    // Every team of the block makes the same number of turns (a barrier inside).
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * block_rows; base < a.rows;
         base += step) {
        const int64_t row = base + team.index * place.rows + place.row;
        const bool live = row < a.rows;  // the block's last teams may have no row
        const int hidden = live ? a.hidden : 0;
        const int64_t first = row * a.hidden;
        const X* x = static_cast<const X*>(a.x) + row * a.x_stride;
        int column[V];
        float u[V][N];
        Raw<X, N> raw_x[V];
        float weight[V][N];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            column[v] = ((v * a.parts + team.part) * kWave + place.lane) * N;
            raw_x[v] = load<kAccess, X, N>(x, column[v], hidden);
        }
        if constexpr (kBranch) {
            const B* branch = static_cast<const B*>(a.branch) + row * a.branch_stride;
            Raw<B, N> raw_branch[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                raw_branch[v] = load<kAccess, B, N>(branch, column[v], hidden);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                load_weight<kAccess, N>(a.weight, a.weight_dtype, column[v], hidden, weight[v]);
            }
            X* updated = static_cast<X*>(a.updated) + first;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float added[N];
                settle<kAccess>(raw_x[v], column[v], hidden);
                settle<kAccess>(raw_branch[v], column[v], hidden);
                widen<X, N>(raw_x[v], u[v]);
                widen<B, N>(raw_branch[v], added);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    u[v][e] += added[e];
                }
                // The norm is taken of the rounded stream, which is what the
                // backward and the next layer read.
                const Raw<X, N> rounded = narrow<X, N>(u[v]);
                store<kAccess, kForwardStores, X, N>(updated, column[v], hidden, rounded);
                widen<X, N>(rounded, u[v]);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                load_weight<kAccess, N>(a.weight, a.weight_dtype, column[v], hidden, weight[v]);
                settle<kAccess>(raw_x[v], column[v], hidden);
                widen<X, N>(raw_x[v], u[v]);
            }
        }

        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                sum += u[v][e] * u[v][e];
            }
        }
        sum = kAccess == Access::kLanes ? lanes_sum(sum, a.row_lanes) : wave_sum(sum);
        // The 8-bit steps' values: u itself for the checkpoint, u * weight for codes.
        uint32_t maximum[V];
        const bool whole_row = kMode == Mode::kQuantize && a.groups == 1;
        if constexpr (kMode != Mode::kNormalize) {
            if constexpr (kMode == Mode::kQuantize) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        u[v][e] *= weight[v][e];
                    }
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                maximum[v] = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    maximum[v] = larger(maximum[v], magnitude_bits(u[v][e]));
                }
            }
            if (whole_row) {
                uint32_t whole = maximum[0];
#pragma unroll
                for (int v = 1; v < V; ++v) {
                    whole = larger(whole, maximum[v]);
                }
                whole = lanes_max(whole, kAccess == Access::kLanes ? a.row_lanes : kWave);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    maximum[v] = whole;
                }
            } else {
                int lanes = kMode == Mode::kCheckpoint ? kCheckpointGroup / N
                                                       : (1 << a.group_shift) / N;
                if (kAccess == Access::kLanes && a.row_lanes < lanes) {
                    lanes = a.row_lanes;  // the lanes past it hold another row
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    maximum[v] = lanes_max(maximum[v], lanes);
                }
            }
        }
        if (a.parts > 1) {
            // Two buffers: a team's next turn writes the other one while slower
            // waves still read this one.
            sums[turn][team.wave] = sum;
            if (whole_row) {
                maxima[turn][team.wave] = maximum[0];
            }
            __syncthreads();
            const int begin = team.index * a.parts;
            sum = 0.0f;
            for (int part = 0; part < a.parts; ++part) {
                sum += sums[turn][begin + part];
            }
            if (whole_row) {
                uint32_t whole = 0;
                for (int part = 0; part < a.parts; ++part) {
                    whole = larger(whole, maxima[turn][begin + part]);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    maximum[v] = whole;
                }
            }
            turn ^= 1;
        }
        const float rstd = 1.0f / __builtin_sqrtf(sum * a.inv_hidden + a.eps);
        if (kMode != Mode::kQuantize && a.rstd != nullptr && live && team.part == 0 &&
            place.lane == 0) {
            a.rstd[row] = rstd;
        }
        if constexpr (kMode == Mode::kQuantize) {
            const bool e4m3 = a.output_dtype == RLN_DTYPE_E4M3;
            const float top = e4m3 ? 448.0f : 127.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const GroupScale scale = group_scale(maximum[v], top);
                const int group = column[v] >> a.group_shift;
                if (column[v] < hidden && group << a.group_shift == column[v]) {
                    a.scale[row * a.groups + group] = scale.step * rstd;
                }
                float steps[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    steps[e] = u[v][e] * scale.inverse;
                }
                store<kAccess, kForwardStores, int8_t, N>(
                    static_cast<int8_t*>(a.normalized) + first, column[v], hidden,
                    e4m3 ? narrow_e4m3<N>(steps) : narrow_int8<N>(steps));
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (kMode == Mode::kCheckpoint) {
                    const GroupScale scale = group_scale(maximum[v], 127.0f);
                    if (column[v] < hidden && column[v] % kCheckpointGroup == 0) {
                        a.scale[row * a.groups + column[v] / kCheckpointGroup] = scale.step;
                    }
                    float steps[N];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        steps[e] = u[v][e] * scale.inverse;
                    }
                    store<kAccess, kForwardStores, int8_t, N>(
                        a.checkpoint + first, column[v], hidden, narrow_int8<N>(steps));
                }
                float normalized[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    normalized[e] = u[v][e] * rstd * weight[v][e];
                }
                store_as<kAccess, kForwardStores, N>(a.normalized, a.output_dtype, first,
                                                     column[v], hidden, normalized);
            }
        }
    }
}

// ----------------------------------------------------------------------------
// Backward, in two forms; neither uses atomics, both give the same bits on every
// run.
//
// Walk: a block's teams walk the rows block by block; each lane keeps its
// columns' share of the weight's gradient in registers, the block adds its
// teams' shares through LDS and writes them to its row of the partials, which
// reduce_kernel adds in a fixed order.
//
// Slabs, for small launches, whose rows stay in the caches: each team takes one
// row, and the launch's first blocks sum the weight's gradient, each over all rows
// of a slab of columns, from a second reading. One launch and no workspace.

constexpr int kSlabLanes = 4;  // 64 bytes of the stream per row
template <typename X>
constexpr int kSlabColumns = kSlabLanes * kColumns<X>;

template <typename X, typename Y, bool Checkpoint>
__device__ __forceinline__ void sum_slab(const BackwardArgs& a) {
    constexpr int N = kColumns<X>;
    constexpr int kRows = 4;  // rows in flight per thread
    __shared__ float totals[kMaxParts][kSlabColumns<X>];
    const int groups = static_cast<int>(blockDim.x) / kSlabLanes;
    const int place = threadIdx.x % kSlabLanes * N;
    const int column = static_cast<int>(blockIdx.x) * kSlabColumns<X> + place;
    float total[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        total[e] = 0.0f;
    }
    for (int64_t base = threadIdx.x / kSlabLanes; base < a.rows;
         base += static_cast<int64_t>(groups) * kRows) {
        Raw<Y, N> raw_y[kRows];
        Raw<X, N> raw_u[kRows];
        Raw<int8_t, N> raw_kept[kRows];
        float scale[kRows];
        float kept_step[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t row = base + static_cast<int64_t>(k) * groups;
            const int hidden = row < a.rows ? a.hidden : 0;
            raw_y[k] = load<Access::kLanes, Y, N, kCached>(
                static_cast<const Y*>(a.grad_normalized) + row * a.hidden, column, hidden);
            if constexpr (Checkpoint) {
                raw_kept[k] = load<Access::kLanes, int8_t, N, kCached>(
                    a.checkpoint + row * a.hidden, column, hidden);
                kept_step[k] = column < hidden
                    ? a.scale[row * a.groups + column / kCheckpointGroup] : 0.0f;
            } else {
                raw_u[k] = load<Access::kLanes, X, N, kCached>(
                    static_cast<const X*>(a.updated) + row * a.updated_stride, column, hidden);
            }
            scale[k] = hidden > 0 ? a.rstd[row] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int hidden = base + static_cast<int64_t>(k) * groups < a.rows ? a.hidden : 0;
            float upstream[N];
            float unit[N];
            settle<Access::kLanes>(raw_y[k], column, hidden);
            widen<Y, N>(raw_y[k], upstream);
            if constexpr (Checkpoint) {
                settle<Access::kLanes>(raw_kept[k], column, hidden);
                widen<int8_t, N>(raw_kept[k], unit);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    unit[e] *= kept_step[k];
                }
            } else {
                settle<Access::kLanes>(raw_u[k], column, hidden);
                widen<X, N>(raw_u[k], unit);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                total[e] += upstream[e] * (unit[e] * scale[k]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
#pragma unroll
        for (int other = kSlabLanes; other < kWave; other *= 2) {
            total[e] += __shfl_xor(total[e], other);
        }
    }
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave < kSlabLanes) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            totals[wave][place + e] = total[e];
        }
    }
    __syncthreads();
    const int own = blockIdx.x * kSlabColumns<X> + static_cast<int>(threadIdx.x);
    if (threadIdx.x < kSlabColumns<X> && own < a.hidden) {
        float sum = 0.0f;
        for (int other = 0; other < static_cast<int>(blockDim.x) / kWave; ++other) {
            sum += totals[other][threadIdx.x];
        }
        store_one(a.grad_weight, a.weight_dtype, own, sum);
    }
}

template <typename X, typename Y, int V, bool Checkpoint, Access kAccess, bool kSlabs>
__global__ __launch_bounds__(kMaxParts * kWave) void backward_kernel(BackwardArgs a) {
    constexpr int N = kColumns<X>;
    // What a slab block reads again stays cached.
    constexpr int kPolicy = kSlabs ? kCached : kOnce;
    const int slabs = kSlabs ? a.slabs : 0;
    if constexpr (kSlabs) {
        if (static_cast<int>(blockIdx.x) < slabs) {
            sum_slab<X, Y, Checkpoint>(a);
            return;
        }
    }
    extern __shared__ float shares[];  // [teams - 1][hidden], the weight's gradient
    __shared__ float sums[2][kMaxParts];
    const Team team = team_of(a.parts);
    const Place place = place_of<kAccess>(a.row_lanes);
    const int block_rows = team.teams * place.rows;
    int column[V];
    float weight[V][N];
    float grad_weight[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        column[v] = ((v * a.parts + team.part) * kWave + place.lane) * N;
        load_weight<kAccess, N>(a.weight, a.weight_dtype, column[v], a.hidden, weight[v]);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            grad_weight[v][e] = 0.0f;
        }
    }
    const int64_t step = (static_cast<int64_t>(gridDim.x) - slabs) * block_rows;
    int turn = 0;
    // Every team of the block makes the same number of turns (barriers inside).
    for (int64_t base = (static_cast<int64_t>(blockIdx.x) - slabs) * block_rows; base < a.rows;
         base += step) {
        const int64_t row = base + team.index * place.rows + place.row;
        const bool live = row < a.rows;
        const int hidden = live ? a.hidden : 0;
        const int64_t first = row * a.hidden;
        Raw<Y, N> raw_y[V];
        Raw<X, N> raw_u[V];
        Raw<int8_t, N> raw_kept[V];
        float kept_step[V];
        Raw<X, N> raw_grad[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            raw_y[v] = load<kAccess, Y, N, kPolicy>(
                static_cast<const Y*>(a.grad_normalized) + first, column[v], hidden);
            if constexpr (Checkpoint) {
                raw_kept[v] = load<kAccess, int8_t, N, kPolicy>(a.checkpoint + first, column[v],
                                                               hidden);
                kept_step[v] = column[v] < hidden
                    ? a.scale[row * a.groups + column[v] / kCheckpointGroup] : 0.0f;
            } else {
                raw_u[v] = load<kAccess, X, N, kPolicy>(
                    static_cast<const X*>(a.updated) + row * a.updated_stride, column[v], hidden);
            }
        }
        if (a.grad_updated != nullptr) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                raw_grad[v] = load<kAccess, X, N>(static_cast<const X*>(a.grad_updated) + first,
                                                  column[v], hidden);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int i = 0; i < Raw<X, N>::kWords; ++i) {
                    raw_grad[v].words[i] = 0;
                }
            }
        }
        const float rstd = live ? a.rstd[row] : 0.0f;
        float unit[V][N];
        float product[V][N];
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float upstream[N];
            settle<kAccess>(raw_y[v], column[v], hidden);
            widen<Y, N>(raw_y[v], upstream);
            if constexpr (Checkpoint) {
                settle<kAccess>(raw_kept[v], column[v], hidden);
                widen<int8_t, N>(raw_kept[v], unit[v]);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    unit[v][e] *= kept_step[v];
                }
            } else {
                settle<kAccess>(raw_u[v], column[v], hidden);
                widen<X, N>(raw_u[v], unit[v]);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                unit[v][e] *= rstd;
                product[v][e] = upstream[e] * weight[v][e];
                sum += product[v][e] * unit[v][e];
                if constexpr (!kSlabs) {
                    grad_weight[v][e] += upstream[e] * unit[v][e];
                }
            }
        }
        sum = kAccess == Access::kLanes ? lanes_sum(sum, a.row_lanes) : wave_sum(sum);
        if (a.parts > 1) {
            // Two buffers: a team's next turn writes the other one while
            // slower waves still read this one.
            sums[turn][team.wave] = sum;
            __syncthreads();
            const int begin = team.index * a.parts;
            sum = 0.0f;
            for (int part = 0; part < a.parts; ++part) {
                sum += sums[turn][begin + part];
            }
            turn ^= 1;
        }
        const float shared = sum * a.inv_hidden;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float gradient[N];
            settle<kAccess>(raw_grad[v], column[v], hidden);
            widen<X, N>(raw_grad[v], gradient);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                gradient[e] += rstd * (product[v][e] - unit[v][e] * shared);
            }
            store<kAccess, kBackwardStores, X, N>(static_cast<X*>(a.grad_x) + first, column[v],
                                                  hidden, narrow<X, N>(gradient));
            if (a.grad_branch != nullptr) {
                store_as<kAccess, kBackwardStores, N>(a.grad_branch, a.branch_dtype, first,
                                                      column[v], hidden, gradient);
            }
        }
    }
    if (kSlabs || a.partials == nullptr) {
        return;
    }
    if constexpr (kAccess == Access::kLanes) {
        // The wave's rows first; row 0's lanes stand for all of them.
#pragma unroll
        for (int e = 0; e < N; ++e) {
            for (int other = a.row_lanes; other < kWave; other *= 2) {
                grad_weight[0][e] += __shfl_xor(grad_weight[0][e], other);
            }
        }
        if (place.row > 0) {
            column[0] = a.hidden;  // past the end: nothing to leave or to store
        }
    }
    // Teams 1, 2, ... leave their shares; team 0 adds them in that order.
    if (team.index > 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (column[v] + e < a.hidden) {
                    shares[(team.index - 1) * a.hidden + column[v] + e] = grad_weight[v][e];
                }
            }
        }
    }
    if (team.teams > 1) {
        __syncthreads();
    }
    if (team.index == 0) {
        float* partial = a.partials + static_cast<int64_t>(blockIdx.x) * a.hidden;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            for (int other = 0; other < team.teams - 1; ++other) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (column[v] + e < a.hidden) {
                        grad_weight[v][e] += shares[other * a.hidden + column[v] + e];
                    }
                }
            }
            store<kAccess, kBackwardStores, float, N>(partial, column[v], a.hidden,
                                                      narrow<float, N>(grad_weight[v]));
        }
    }
}

// ----------------------------------------------------------------------------
// Launch shapes (host). Measured on MI355X, graphs of launches over buffers that
// pass the caches, TB/s of algorithmic bytes (a large copy reaches 5.4):
//
//  * 16 bytes of the stream per lane and slot. The forward takes one slot of a
//    16-bit stream ([16384, 4096] bf16: 6.2 against 5.9 with two) and two of a
//    32-bit one, whose half as many waves then store whole words of codes
//    ([32768, 1024] e4m3 in fp32: 6.2 against 5.4 with one; without codes 6.2
//    against 5.9), and doubles them until a row fits 8 waves, a 32-bit stream's up
//    to four: in blocks of 16 waves a CU idles while they wait for each other
//    ([8192, 8192] fp32 with the checkpoint: 5.6 with four slots and 8 waves, 5.2
//    with two and 16). A 16-bit stream's stop at two, so that its rows past 8192
//    columns take 9 to 16 waves, at no loss ([8192, 16384] bf16: 6.0, [8192, 9216]
//    6.0, [8192, 8192] in 8 waves 6.0).
//  * Short rows share waves, 2, 4 or 8 in each ([262144, 128] bf16 forward 52 against
//    83 us with a wave for each, with codes 44 against 110, backward 50 against 80;
//    [524288, 64] 52 against 156, 71 with at least 16 lanes a row).
//  * The backward holds the weight and its gradient's sums in registers besides
//    and takes one slot up to 8 waves a row ([32768, 1024] fp32: 5.7 against 5.4
//    with two). Longer 32-bit rows take two up to 16 waves ([8192, 8192]: 5.5
//    against 5.2 with four and 8 waves).
//  * Its grid is two blocks of about 8 waves for each CU, or one of more: the same
//    number everywhere, since blocks walk the rows at one pace ([6553, 5120] bf16:
//    52 us with two blocks of 5 waves per CU, 61 with three), and no more, since
//    each adds a row of partial sums ([16384, 4096] bf16: 90 us at 16 waves per CU,
//    104 at 8, 104 at 32).
//  * Slab blocks sum the weight's gradient of launches of up to 1024 rows and 2^21
//    elements, whose time is launches more than bytes: [256, 384] fp32 3.5 against
//    6.0 us for the walk and its reduction, [1024, 768] 7.1 against 9.5, [512, 4096]
//    bf16 8.3 against 12.6. Past that their second reading costs more: [2048, 2048]
//    bf16 15.3 against 14.1, [4096, 384] fp32 17.1 against 11.4.
//  * Decode-sized forwards, at most a row for each CU, wait for one row's chain of
//    steps: one slot up to 12 waves ([64, 5120] bf16 e4m3: 4.1 against 4.4 us,
//    [256, 2048] fp32 3.5 against 3.8), longer rows as above ([8, 4096] fp32:
//    3.1 with two slots, 3.5 with one and 16 waves).

constexpr int64_t kComputeUnits = 256;

struct Shape {
    int slots;  // V
    int parts;
    int threads;
    int row_lanes;  // below 64: several rows per wave
};

inline int columns_of(int dtype) {
    return dtype == RLN_DTYPE_F32 ? 4 : 8;
}

// Waves that one slot per lane needs for a row.
inline int64_t wave_vectors(int64_t hidden, int x_dtype) {
    const int columns = columns_of(x_dtype) * kWave;
    return (hidden + columns - 1) / columns;
}

// Waves per row at `slots` vectors per lane, and teams that make blocks of about
// `waves` waves (nearest; at least one team).
inline Shape shape_of(int64_t vectors, int slots, int waves) {
    Shape shape;
    shape.row_lanes = kWave;
    shape.slots = slots;
    shape.parts = static_cast<int>((vectors + slots - 1) / slots);
    const int teams = (waves + shape.parts / 2) / shape.parts;
    shape.threads = (teams > 1 ? teams : 1) * shape.parts * kWave;
    return shape;
}

inline int teams_of(const Shape& shape) {
    return shape.threads / (kWave * shape.parts);
}

// Blocks that give every row its lanes (no overflow for any row count).
inline int64_t blocks_of(int64_t rows, const Shape& shape) {
    const int block_rows = teams_of(shape) * (kWave / shape.row_lanes);
    return rows / block_rows + (rows % block_rows != 0);
}

// Rows of at most half a wave's columns share waves: 2, 4 or 8 in each.
inline Shape short_shape(int64_t hidden, int x_dtype, int waves) {
    const int columns = columns_of(x_dtype);
    Shape shape = shape_of(1, 1, waves);
    shape.row_lanes = hidden <= 8 * columns ? 8 : hidden <= 16 * columns ? 16 : 32;
    return shape;
}

inline Shape forward_shape(int64_t rows, int64_t hidden, int x_dtype) {
    if (hidden <= 32 * columns_of(x_dtype)) {
        return short_shape(hidden, x_dtype, 4);
    }
    const int64_t vectors = wave_vectors(hidden, x_dtype);
    if (rows <= kComputeUnits && vectors <= 12) {
        return shape_of(vectors, 1, 4);
    }
    const int most = x_dtype == RLN_DTYPE_F32 ? 4 : 2;
    int slots = x_dtype == RLN_DTYPE_F32 && vectors > 1 ? 2 : 1;
    while (slots < most && slots * 8 < vectors) {
        slots *= 2;
    }
    return shape_of(vectors, slots, 4);
}

constexpr int64_t kMaxBlocks = 1 << 21;

inline int64_t forward_blocks(int64_t rows, const Shape& shape) {
    const int64_t blocks = blocks_of(rows, shape);
    return blocks < kMaxBlocks ? blocks : kMaxBlocks;
}

inline Shape backward_shape(int64_t hidden, int x_dtype) {
    if (hidden <= 32 * columns_of(x_dtype)) {
        return short_shape(hidden, x_dtype, 8);
    }
    const int64_t vectors = wave_vectors(hidden, x_dtype);
    const int slots = vectors <= 8 ? 1 : vectors <= 2 * kMaxParts ? 2 : 4;
    return shape_of(vectors, slots, 8);
}

constexpr int64_t kSlabRows = 1024;
constexpr int64_t kSlabElements = 1 << 21;

inline bool backward_slabs(int64_t rows, int64_t hidden) {
    return rows <= kSlabRows && rows * hidden <= kSlabElements;
}

inline int64_t backward_blocks(int64_t rows, const Shape& shape) {
    const int64_t blocks = blocks_of(rows, shape);
    const int64_t most = shape.threads <= 10 * kWave ? 2 * kComputeUnits : kComputeUnits;
    return blocks < most ? blocks : most;
}

// Defined in rms_kernels.hip, one translation unit per stream type and pass.
template <typename X>
int launch_forward(const ForwardArgs& a, const Shape& shape, int branch_dtype, Mode mode,
                   hipStream_t stream);
template <typename X>
int launch_backward(const BackwardArgs& a, const Shape& shape, int grad_dtype,
                    hipStream_t stream);

}  // namespace rms
}  // namespace rln

#endif  // RMS_DEVICE_H
