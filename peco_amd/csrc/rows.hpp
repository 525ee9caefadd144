// Rows of channels spread over the lanes of part of a wavefront, of one or of several, for the kernels that take
// statistics over a row (layer norm, its gradient, quantization).
//
// A row of C channels is held in registers by `lanes` lanes, kChunks pieces of 8 adjacent channels each, whatever the
// rows' alignment: 16-byte accesses may start at any element. Short rows share a wavefront; those of one wavefront need no
// barrier for their sums.
#pragma once

#include "mfma.hpp"

#include <type_traits>

namespace peco {

constexpr int kMaxRowChannels = 8 * kWave * 8 * 4;

// Where the rows of a tensor [n0, n1, n2, C] lie (strides in elements; channels adjacent).
struct RowMap {
    int64_t s0, s1, s2;
    uint32_t n1, n2;
    int flat;  // one distance s2 between all rows
    __device__ __forceinline__ int64_t at(uint32_t row) const {
        if (flat) return row * s2;
        const uint32_t a = row / n2, c = row - a * n2;
        const uint32_t e = a / n1, b = a - e * n1;
        return e * s0 + b * s1 + c * s2;
    }
};

inline RowMap row_map(const int64_t* strides, int n0, int n1, int n2) {
    RowMap m{strides[0], strides[1], strides[2], static_cast<uint32_t>(n1), static_cast<uint32_t>(n2), 0};
    if (n2 == 1) m.s2 = n1 == 1 ? m.s0 : m.s1;  // the distance between the rows of the innermost axis that has some
    const bool inner = n1 == 1 || n2 == 1 || m.s1 == n2 * m.s2;
    const int64_t row = static_cast<int64_t>(n1) * n2;
    m.flat = inner && (n0 == 1 || m.s0 == row * m.s2);
    return m;
}

// Eight channels as they lie in memory. (Words, not 16-bit elements: the compiler would keep each of those in a register
// of its own across a loop.)
template <int DT> struct Piece {
    static constexpr int kWords = DT == kF32 ? 8 : 4;
    uint32_t word[kWords];
    typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));  // at any element
    // (A row's start, the same in a wavefront that has one row, and a 32-bit offset: one register for the address.)
    __device__ __forceinline__ void load(const char* row, uint32_t column) {
        const Any* p = reinterpret_cast<const Any*>(row + column * (DT == kF32 ? 4u : 2u));
#pragma unroll
        for (int j = 0; j < kWords / 4; ++j) {
            const Any v = p[j];
#pragma unroll
            for (int k = 0; k < 4; ++k) word[4 * j + k] = v[k];
        }
    }
    __device__ __forceinline__ void store(char* row, uint32_t column) const {
        Any* p = reinterpret_cast<Any*>(row + column * (DT == kF32 ? 4u : 2u));
#pragma unroll
        for (int j = 0; j < kWords / 4; ++j) p[j] = Any{word[4 * j], word[4 * j + 1], word[4 * j + 2], word[4 * j + 3]};
    }
    __device__ __forceinline__ uint32_t bits(int k) const {
        return DT == kF32 ? word[k] : k % 2 ? word[k / 2] >> 16 : word[k / 2] & 0xffffu;
    }
    // The channels moved `by` (0 to 8) places down, 0 behind them.
    __device__ __forceinline__ void shift(int by) {
        constexpr int kPer = DT == kF32 ? 1 : 2;  // channels a word
#pragma unroll
        for (int step = 8; step >= kPer; step /= 2)
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const int from = j + step / kPer;
                word[j] = by & step ? from < kWords ? word[from] : 0u : word[j];
            }
        if constexpr (kPer == 2)
#pragma unroll
            for (int j = 0; j < kWords; ++j)
                word[j] = by & 1 ? word[j] >> 16 | (j + 1 < kWords ? word[j + 1] << 16 : 0u) : word[j];
    }
    __device__ __forceinline__ float get(int k) const {
        if constexpr (DT == kF32) return __uint_as_float(word[k]);
        else if constexpr (DT == kBF16) return __uint_as_float(k % 2 ? word[k / 2] & 0xffff0000u : word[k / 2] << 16);
        else return f16_bits_to_f32(static_cast<uint16_t>(k % 2 ? word[k / 2] >> 16 : word[k / 2]));
    }
    // Makes the compiler take the values from the words again where it would keep them.
    __device__ __forceinline__ void again() {
        if constexpr (DT != kF32)
#pragma unroll
            for (int j = 0; j < kWords; ++j) asm("" : "+v"(word[j]));
    }
};

// The lanes of one row: lane of lanes, and the row's length.
struct RowLanes {
    int lane, lanes, channels;
    __device__ __forceinline__ int first(int c) const { return (c * lanes + lane) * 8; }
    // Whether element k of piece c lies in the row (kWhole: its length is a multiple of 8).
    template <bool kWhole> __device__ __forceinline__ bool inside(int c, int k) const {
        return first(c) + (kWhole ? 0 : k) < channels;
    }
};

// A lane's pieces of the row at `offset` (elements), 0 behind the row's end: the 8 channels before it are taken for a
// piece that meets it, and moved.
template <int DT, bool kWhole, int kChunks>
__device__ __forceinline__ void load_row(Piece<DT> (&x)[kChunks], const void* base, int64_t offset, const RowLanes& r) {
    const char* row = static_cast<const char*>(base) + offset * (DT == kF32 ? 4 : 2);
    if (!kWhole && r.channels < 8) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) x[c] = Piece<DT>{};
        if (r.lane == 0)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < r.channels) {
                    if constexpr (DT == kF32) x[0].word[k] = reinterpret_cast<const uint32_t*>(row)[k];
                    else x[0].word[k / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k]) << (k % 2 * 16);
                }
        return;
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) x[c].load(row, min(r.first(c), r.channels - 8));  // all in flight
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        if constexpr (kWhole) {
#pragma unroll
            for (int k = 0; k < Piece<DT>::kWords; ++k) x[c].word[k] = r.first(c) < r.channels ? x[c].word[k] : 0;
        } else {
            x[c].shift(min(max(r.first(c) - (r.channels - 8), 0), 8));
        }
    }
}

// Eight fp32 values rounded to the type.
template <int DT> __device__ __forceinline__ Piece<DT> round_piece(const float (&v)[8]) {
    Piece<DT> y;
#pragma unroll
    for (int k = 0; k < Piece<DT>::kWords; ++k) {
        if constexpr (DT == kF32) y.word[k] = __float_as_uint(v[k]);
        else y.word[k] = Mfma<DT>::pack2(v[2 * k], v[2 * k + 1]);
    }
    return y;
}

template <int DT, bool kWhole>
__device__ __forceinline__ void store_piece(const Piece<DT>& y, void* base, int64_t offset, int c, const RowLanes& r) {
    char* row = static_cast<char*>(base) + offset * (DT == kF32 ? 4 : 2);
    const int col = r.first(c);
    if (col + (kWhole ? 0 : 7) < r.channels) {
        y.store(row, col);
    } else if (!kWhole) {
#pragma unroll
        for (int k = 0; k < 7; ++k) {
            if (col + k >= r.channels) break;
            if constexpr (DT == kF32) reinterpret_cast<uint32_t*>(row)[static_cast<uint32_t>(col + k)] = y.bits(k);
            else reinterpret_cast<uint16_t*>(row)[static_cast<uint32_t>(col + k)] = static_cast<uint16_t>(y.bits(k));
        }
    }
}

// A lane's pieces of a weight or bias (of the rows' type, or fp32) as fp32, 0 behind the row's end.
template <int DT, bool kWhole, int kChunks>
__device__ __forceinline__ void load_weight(float (&w)[kChunks][8], const void* base, int64_t offset, bool wide,
                                            const RowLanes& r) {
    if (DT == kF32 || wide) {
        Piece<kF32> x[kChunks];
        load_row<kF32, kWhole>(x, base, offset, r);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[c][k] = x[c].get(k);
    } else {
        Piece<DT> x[kChunks];
        load_row<DT, kWhole>(x, base, offset, r);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[c][k] = x[c].get(k);
    }
}

struct AddF {
    static __device__ __forceinline__ uint32_t run(uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }
};
struct MaxU {
    static __device__ __forceinline__ uint32_t run(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// v combined over groups of L adjacent lanes, the same in all of them: pairs, quads (quad_perm), then the mirrored lane
// of 8 and of 16, and the wavefront's quarters and halves.
template <typename Op, int L> __device__ __forceinline__ uint32_t combine_lanes(uint32_t v) {
    v = Op::run(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, false));
    v = Op::run(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, false));
    if constexpr (L > 4) v = Op::run(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false));
    if constexpr (L > 8) v = Op::run(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, false));
    if constexpr (L > 16) v = Op::run(v, wave_shfl_xor(v, 16));
    if constexpr (L > 32) v = Op::run(v, wave_shfl_xor(v, 32));
    return v;
}

// The same over rows of `waves` whole wavefronts (every wavefront of the workgroup calls it the same number of times).
// slots: 2 x 16 words of LDS, used in turn, so that one barrier a call is enough: a wavefront that writes a half again
// has passed the barrier of the call between, before which every wavefront had read it.
template <int L> struct RowCombine {
    uint32_t (*slots)[16];
    int waves, wave, half = 0;
    template <typename Op> __device__ __forceinline__ uint32_t run(uint32_t v) {
        v = combine_lanes<Op, L>(v);
        if (L < kWave || waves == 1) return v;
        slots[half][wave] = v;
        __syncthreads();
        const int first = wave / waves * waves;
        v = slots[half][first];
        for (int i = 1; i < waves; ++i) v = Op::run(v, slots[half][first + i]);
        half ^= 1;
        return v;
    }
    __device__ __forceinline__ float sum(float v) { return __uint_as_float(run<AddF>(__float_as_uint(v))); }
    __device__ __forceinline__ void sum2(float& a, float& b) {
        uint32_t u = combine_lanes<AddF, L>(__float_as_uint(a)), v = combine_lanes<AddF, L>(__float_as_uint(b));
        if (L == kWave && waves > 1) {
            slots[half][wave] = u;
            slots[half][8 + wave] = v;
            __syncthreads();
            const int first = wave / waves * waves;
            u = slots[half][first];
            v = slots[half][8 + first];
            for (int i = 1; i < waves; ++i) {
                u = AddF::run(u, slots[half][first + i]);
                v = AddF::run(v, slots[half][8 + first + i]);
            }
            half ^= 1;
        }
        a = __uint_as_float(u);
        b = __uint_as_float(v);
    }
};

// A row's scale and codes from the bits of its largest magnitude (whose order is that of the magnitudes, with NaN above
// infinity): see norm.hip.
struct RowScale {
    float most, by;
    bool finite, zero;
    __device__ __forceinline__ explicit RowScale(uint32_t bits)
        : most(__uint_as_float(bits)), finite(bits < 0x7f800000u), zero(most < 127.0f * 0x1p-126f) {
        by = finite && !zero ? 127.0f * (1.0f / most) : 0.0f;
    }
    __device__ __forceinline__ float scale() const {
        return !finite ? __uint_as_float(0x7fc00000u) : zero ? 0.0f : most * (1.0f / 127.0f);
    }
    __device__ __forceinline__ int code(float x) const { return finite ? static_cast<int>(rintf(x * by)) : 0; }
};

// What the norm keeps of a row: its mean in two parts, and 1 / sqrt(variance + eps).
struct RowStats {
    float mean, rest, inverse;
};

// The number of a lane's row among the workgroup's.
template <int L> __device__ __forceinline__ uint32_t row_in_group(int row_lanes) {
    const uint32_t row = threadIdx.x / row_lanes;
    return L == kWave ? __builtin_amdgcn_readfirstlane(row) : row;
}

// How rows of C channels are spread: lanes of a wavefront, pieces a lane, wavefronts a row, and rows and threads of a
// workgroup of at most `most_waves`. Rows of more than a wavefront take as many as hold them with `most_chunks` pieces
// a lane, or with more where 8 do not.
struct RowShape {
    int lanes, chunks, waves, threads, rows;
};
inline RowShape row_shape(int channels, int most_chunks, int most_waves) {
    RowShape s{kWave, 1, 1, 0, 0};
    if (channels <= 64) s.lanes = 8;
    else if (channels <= 128) s.lanes = 16;
    while (s.chunks < most_chunks && s.lanes * s.chunks * 8 < channels) s.chunks *= 2;
    while (s.chunks < 4 && 8 * s.lanes * s.chunks * 8 < channels) s.chunks *= 2;
    s.waves = static_cast<int>(ceil_div(channels, s.lanes * s.chunks * 8));
    if (s.waves > most_waves) most_waves = 8;
    s.rows = s.lanes < kWave ? most_waves * (kWave / s.lanes) : most_waves / s.waves;
    s.threads = s.rows * s.waves * s.lanes;
    return s;
}

// Rows [n0, n1, n2] of x quantized: codes int8 (rows `pitch` bytes apart) and a scale a row (norm.hip).
int launch_quantize_rows(const void* x, const int64_t* strides, int8_t* codes, int64_t pitch, float* scales, int n0,
                         int n1, int n2, int channels, int dtype, hipStream_t stream);

}  // namespace peco
