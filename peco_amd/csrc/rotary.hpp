// Rotary positions with several axes: the angles of a row's channel pairs from its positions.
//
// Pair i belongs to one axis (time, height, width, ...) and turns by position[axis] * frequency_i. The
// frequencies come as turns per unit of position (frequency / 2 pi) in 64 bits, and the product is taken
// to its fraction of a turn in 64 bits too: in 32 bits a position of 2^17 would leave an angle 2^-7 radians
// off. Sine and cosine of the fraction are then taken in 32 bits. The few 64-bit operations are spent once
// per row and pair and shared by the heads a lane turns.
#pragma once

#include "common.hpp"

namespace peco {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 128;

enum PositionType : int { kPosI32 = 0, kPosI64 = 1, kPosF32 = 2 };

struct RotaryPlan {
    double turns[kMaxPairs];  // turns per unit of position of each pair
    const void* positions;    // [batch, axes, rows], rows adjacent
    int64_t batch_stride, axis_stride;
    int type;
    int axes;
    int bound[kMaxAxes];      // pairs below bound[a] belong to the axes up to a
    int pairs;                // pairs that turn; the channels behind them are copied
    float sign;               // -1: the inverse rotation
};

// Fills the plan; false for arguments that the kernels do not take. `turns` [sum of axis_pairs] and
// `axis_pairs` [axes] are host memory.
inline bool make_plan(RotaryPlan& p, const void* positions, int type, int64_t batch_stride, int64_t axis_stride,
                      const double* turns, const int* axis_pairs, int axes, int halves, int inverse, int dims) {
    if (!positions || !turns || !axis_pairs || axes < 1 || axes > kMaxAxes || type < 0 || type > kPosF32) return false;
    int pairs = 0;
    for (int a = 0; a < axes; ++a) {
        if (axis_pairs[a] < 1 || axis_pairs[a] > kMaxPairs || pairs + axis_pairs[a] > kMaxPairs) return false;
        pairs += axis_pairs[a];
        p.bound[a] = pairs;
    }
    for (int a = axes; a < kMaxAxes; ++a) p.bound[a] = pairs;
    if (2 * pairs > dims || (halves && pairs % 8)) return false;
    for (int i = 0; i < kMaxPairs; ++i) p.turns[i] = i < pairs ? turns[i] : 0.0;
    p.positions = positions;
    p.type = type;
    p.batch_stride = batch_stride;
    p.axis_stride = axis_stride;
    p.axes = axes;
    p.pairs = pairs;
    p.sign = inverse ? -1.0f : 1.0f;
    return true;
}

// Cosine and sine of pairs [first, first + N) of row `row` of batch entry `b`. Pairs past plan.pairs are
// not written (the caller copies their channels).
template <int N>
__device__ __forceinline__ void rotary_angles(const RotaryPlan& p, int b, int64_t row, int first, float (&c)[N],
                                              float (&s)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = first + k;
        c[k] = 1.0f;
        s[k] = 0.0f;
        if (i >= p.pairs) continue;
        const int axis = (i >= p.bound[0]) + (i >= p.bound[1]) + (i >= p.bound[2]);
        const int64_t at = b * p.batch_stride + axis * p.axis_stride + row;
        const double pos = p.type == kPosI32   ? static_cast<double>(static_cast<const int32_t*>(p.positions)[at])
                           : p.type == kPosI64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                               : static_cast<double>(static_cast<const float*>(p.positions)[at]);
        const double t = pos * p.turns[i];
        float sine, cosine;
        sincospif(2.0f * static_cast<float>(t - __builtin_rint(t)), &sine, &cosine);
        c[k] = cosine;
        s[k] = sine * p.sign;
    }
}

// Eight channels as a row holds them, and their values in fp32.
template <int DT> struct Chunk {
    u16x8 raw;
    __device__ __forceinline__ void load(const void* base, int64_t i) {
        raw = *reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(base) + i);
    }
    __device__ __forceinline__ void store(void* base, int64_t i) const {
        *reinterpret_cast<u16x8*>(static_cast<uint16_t*>(base) + i) = raw;
    }
    __device__ __forceinline__ float get(int k) const { return half_to_f32<DT>(raw[k]); }
    __device__ __forceinline__ void set(int k, float v) { raw[k] = f32_to_half<DT>(v); }
};
template <> struct Chunk<kF32> {
    f32x4 raw[2];
    __device__ __forceinline__ void load(const void* base, int64_t i) {
        const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i);
        raw[0] = p[0];
        raw[1] = p[1];
    }
    __device__ __forceinline__ void store(void* base, int64_t i) const {
        f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + i);
        p[0] = raw[0];
        p[1] = raw[1];
    }
    __device__ __forceinline__ float get(int k) const { return raw[k / 4][k % 4]; }
    __device__ __forceinline__ void set(int k, float v) { raw[k / 4][k % 4] = v; }
};

// Adjacent channels (2 k, 2 k + 1) of one chunk turned as pairs `first` + k.
template <int DT>
__device__ __forceinline__ void turn_adjacent(Chunk<DT>& x, int first, int pairs, const float (&c)[4],
                                              const float (&s)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (first + k >= pairs) continue;
        const float a = x.get(2 * k), b = x.get(2 * k + 1);
        x.set(2 * k, a * c[k] - b * s[k]);
        x.set(2 * k + 1, b * c[k] + a * s[k]);
    }
}

}  // namespace peco
