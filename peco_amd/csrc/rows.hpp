// Rows of channels spread over the lanes of part of a wavefront, of one or of several, for the kernels that take
// statistics over a row (layer norm, its gradient, quantization).
//
// A row of C channels is held in registers by `lanes` lanes, kChunks pieces of 8 channels each: adjacent channels
// where everything lies on 16 bytes (kVec), else channels `lanes` apart, so that the single loads of a wavefront are
// adjacent. Rows of up to 512 channels take 8, 16 or 64 lanes with one piece (several rows a wavefront below 64), of up
// to 2048 one wavefront with 1, 2 or 4 pieces, so that their sums need no barrier; longer ones 2, 4 or 8 wavefronts.
#pragma once

#include "mfma.hpp"
#include "rotary.hpp"

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

// Whether every row starts on 16 bytes.
inline bool rows_on_16(const void* p, const int64_t* strides, int size) {
    return !(reinterpret_cast<uintptr_t>(p) % 16) && !(((strides[0] | strides[1] | strides[2]) * size) % 16);
}

// The lanes of one row: lane of lanes, and the row's length.
struct RowLanes {
    int lane, lanes, channels;
    template <bool kVec> __device__ __forceinline__ int first(int c) const {
        return kVec ? (c * lanes + lane) * 8 : c * 8 * lanes + lane;
    }
    template <bool kVec> __device__ __forceinline__ int column(int c, int k) const {
        return first<kVec>(c) + (kVec ? k : k * lanes);
    }
};

// A lane's pieces of the row at `offset` (elements), 0 behind the row's end.
template <int DT, bool kVec, int kChunks>
__device__ __forceinline__ void load_row(Chunk<DT> (&x)[kChunks], const void* base, int64_t offset, const RowLanes& r) {
    if constexpr (kVec) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {  // clamped, unconditional: all loads in flight
            const int col = r.template first<true>(c);
            x[c].load(base, offset + min(col, r.channels - 8));
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            if (r.template first<true>(c) >= r.channels) x[c] = Chunk<DT>{};
    } else {
        using T = std::conditional_t<DT == kF32, float, uint16_t>;
        T v[kChunks][8];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[c][k] = static_cast<const T*>(base)[offset + min(r.template column<false>(c, k), r.channels - 1)];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const T w = r.template column<false>(c, k) < r.channels ? v[c][k] : T{};
                if constexpr (DT == kF32) x[c].raw[k / 4][k % 4] = w;
                else x[c].raw[k] = w;
            }
    }
}

// Eight fp32 values rounded to the type.
template <int DT> __device__ __forceinline__ Chunk<DT> round_chunk(const float (&v)[8]) {
    Chunk<DT> y;
    if constexpr (DT == kF32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) y.raw[k / 4][k % 4] = v[k];
    } else {
        u32x4 p;
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = Mfma<DT>::pack2(v[2 * k], v[2 * k + 1]);
        y.raw = __builtin_bit_cast(u16x8, p);
    }
    return y;
}

template <int DT, bool kVec>
__device__ __forceinline__ void store_piece(const Chunk<DT>& y, void* base, int64_t offset, int c, const RowLanes& r) {
    if constexpr (kVec) {
        const int col = r.template first<true>(c);
        if (col < r.channels) y.store(base, offset + col);
    } else {
        using T = std::conditional_t<DT == kF32, float, uint16_t>;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int col = r.template column<false>(c, k);
            if constexpr (DT == kF32) {
                if (col < r.channels) static_cast<T*>(base)[offset + col] = y.raw[k / 4][k % 4];
            } else {
                if (col < r.channels) static_cast<T*>(base)[offset + col] = y.raw[k];
            }
        }
    }
}

// A lane's pieces of a weight or bias (of the rows' type, or fp32) as fp32, 0 behind the row's end.
template <int DT, bool kVec, int kChunks>
__device__ __forceinline__ void load_weight(float (&w)[kChunks][8], const void* base, int64_t offset, bool wide,
                                            const RowLanes& r) {
    if (DT == kF32 || wide) {
        Chunk<kF32> x[kChunks];
        load_row<kF32, kVec>(x, base, offset, r);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[c][k] = x[c].get(k);
    } else {
        Chunk<DT> x[kChunks];
        load_row<DT, kVec>(x, base, offset, r);
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
// slots: 2 x 8 words of LDS, used in turn, so that one barrier a call is enough: a wavefront that writes a half again
// has passed the barrier of the call between, before which every wavefront had read it.
template <int L> struct RowCombine {
    uint32_t (*slots)[8];
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
};

// A row's scale and codes from the bits of its largest magnitude (whose order is that of the magnitudes, with NaN above
// infinity): see norm.hip.
struct RowScale {
    float most, by;
    bool finite, zero;
    __device__ __forceinline__ explicit RowScale(uint32_t bits)
        : most(__uint_as_float(bits)), finite(bits < 0x7f800000u), zero(most < 127.0f * 0x1p-126f) {
        by = finite && !zero ? 127.0f / most : 0.0f;
    }
    __device__ __forceinline__ float scale() const {
        return !finite ? __uint_as_float(0x7fc00000u) : zero ? 0.0f : most / 127.0f;
    }
    __device__ __forceinline__ int code(float x) const { return finite ? static_cast<int>(rintf(x * by)) : 0; }
};

// How rows of C channels are spread: lanes of a wavefront, pieces a lane, wavefronts a row, threads a workgroup.
struct RowShape {
    int lanes, chunks, waves, threads, rows;  // rows: of a workgroup
};
inline RowShape row_shape(int channels) {
    RowShape s{kWave, 4, 1, 256, 4};
    if (channels <= 64) s.lanes = 8, s.chunks = 1;
    else if (channels <= 128) s.lanes = 16, s.chunks = 1;
    else if (channels <= 512) s.chunks = 1;
    else if (channels <= 1024) s.chunks = 2;
    while (s.waves * s.lanes * s.chunks * 8 < channels) s.waves *= 2;
    if (s.waves == 8) s.threads = 512;
    s.rows = s.threads / (s.lanes * s.waves);
    return s;
}

// Rows [n0, n1, n2] of x quantized: codes int8 (rows `pitch` bytes apart) and a scale a row (norm.hip).
int launch_quantize_rows(const void* x, const int64_t* strides, int8_t* codes, int64_t pitch, float* scales, int n0,
                         int n1, int n2, int channels, int dtype, hipStream_t stream);

}  // namespace peco
