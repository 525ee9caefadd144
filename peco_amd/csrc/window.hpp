// Attention with a sliding window and sinks: what its forward and backward kernels share.
//
// Mask. A query at position p sees key j when j <= p + right and (j >= p - left or j < sinks). Queries and
// keys of a sequence end together: query i of n stands at p = i + keys - n.
//
// Rows. The `group` query heads of one key head are one stream of rows, r = token * group + head in group, so
// a tile of rows reads each K/V tile once for all of them and dK, dV sum over the heads without atomics.
//
// Key stream. The keys some row of a tile of rows sees are a run of sinks [0, a1) and a run [b0, b0 + n):
// stream row r is key r for r < a1, else r + delta (delta = b0 - a1). delta > 0 only when the sinks end
// before the window of every row begins, so in stream rows the mask of a query is
//   r <= H and (r >= W or r < sinks),   H = min(p + right, last key) - delta, W = p - left - delta.
//
// LDS tiles. 64 rows of D channels, row-major, filled by 16-byte direct loads. The 16-byte chunks of a row
// are XOR-swizzled so that both reads of a tile are free of bank conflicts: 16 rows at one chunk (MFMA A
// operand, rows along M) and 4 rows x 32 bytes (transpose read: channels along M).
#pragma once

#include "mfma.hpp"

namespace peco {

constexpr int kWinTile = 64;      // rows of an LDS tile
constexpr int kWinRows = 128;     // query rows of a forward or dQ workgroup, keys of a dK/dV workgroup
constexpr int kUnbounded = 0x40000000;  // left or right without a limit

template <int D> struct WinTile {
    static constexpr int CH = D / 8;                 // 16-byte chunks per row
    static constexpr int kElems = kWinTile * D;
    static constexpr int kWaveRows = kWave / CH;     // rows per wave-wide direct load
    static constexpr int kLoads = kWinTile / (4 * kWaveRows);  // direct loads per wave per tile (4 waves)
    static __device__ __forceinline__ int swz(int row) {
        return CH == 16 ? 4 * (row % 4) + ((row >> 2) & 3) : 4 * ((row >> 1) & 1) + ((row >> 2) & 3);
    }
    // A operand with the tile's rows along M: row, channels 16 s + 8 h .. + 7.
    static __device__ __forceinline__ u16x8 rows(const uint16_t* t, int row, int s, int h) {
        return *reinterpret_cast<const u16x8*>(t + row * D + ((2 * s + h) ^ swz(row)) * 8);
    }
    // A operand with channels along M: channel 32 nb + l % 32, tile rows row0 + 8 t + 4 h + (0..3), t = 0, 1.
    // Source lane r of each 16-lane group points at row r / 4, channels 32 nb + 16 ((l / 16) % 2) + 4 (r % 4).
    static __device__ __forceinline__ u16x8 channels(const uint16_t* t, int row0, int nb, int lane) {
        const int src = lane % 16, d = 32 * nb + 16 * ((lane / 16) % 2) + 4 * (src % 4);
        u32x2 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = row0 + 8 * u + 4 * (lane / 32) + src / 4;
            const uint16_t* a = t + row * D + ((d / 8) ^ swz(row)) * 8 + (d % 8);
            part[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                    (__attribute__((address_space(3))) s16x4*)(a)));
        }
        return __builtin_bit_cast(u16x8, u32x4{part[0][0], part[0][1], part[1][0], part[1][1]});
    }
};

template <int DT> __device__ __forceinline__ bool not_finite(uint16_t b) {
    constexpr uint16_t kExp = DT == kBF16 ? 0x7f80 : 0x7c00;
    return (b & kExp) == kExp;
}

// Whether any of the 32 tile rows from row0 holds an infinity or NaN.
template <int DT, int D>
__device__ __forceinline__ bool tile_not_finite(const uint16_t* t, int row0, int lane) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 32 * D / 8 / kWave; ++i) {
        const u16x8 x = *reinterpret_cast<const u16x8*>(t + row0 * D + (i * kWave + lane) * 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) bad |= not_finite<DT>(x[k]);
    }
    return __any(bad);
}

// acc += (tile rows row0 .. row0 + 31, channels along M) x w, where w holds this lane's column: packed weight
// pairs of rows 8 (i / 4) + 4 h + i % 4.
template <int DT, int D>
__device__ __forceinline__ void add_rows(f32x16 (&acc)[D / 32], const uint16_t* t, int row0, const uint32_t (&w)[8],
                                         int lane) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const u16x8 b = __builtin_bit_cast(u16x8, u32x4{w[4 * kk], w[4 * kk + 1], w[4 * kk + 2], w[4 * kk + 3]});
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
            acc[nb] = Mfma<DT>::run(WinTile<D>::channels(t, row0 + 16 * kk, nb, lane), b, acc[nb]);
    }
}

// The same for a tile with infinities or NaN in rows that some column hides: a hidden row's weight is 0, but 0
// times them is NaN. Each tile row is multiplied by itself and added where seen(row) holds. The kernels come
// here only in a second walk over their tiles, after a first one met such a tile.
template <int DT, int D, typename Seen>
__device__ __forceinline__ void add_rows_seen(f32x16 (&acc)[D / 32], const uint16_t* t, int row0,
                                              const uint32_t (&w)[8], int lane, const Seen& seen) {
    const int h = lane / 32;
#pragma unroll 1
    for (int row = 0; row < 32; ++row) {
        const bool add = seen(row);
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb) {
            f32x16 one{};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u16x8 a = WinTile<D>::channels(t, row0 + 16 * kk, nb, lane);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (16 * kk + 8 * (e / 4) + 4 * h + e % 4 != row) a[e] = 0;
                const u16x8 b =
                    __builtin_bit_cast(u16x8, u32x4{w[4 * kk], w[4 * kk + 1], w[4 * kk + 2], w[4 * kk + 3]});
                one = Mfma<DT>::run(a, b, one);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[nb][i] += add ? one[i] : 0.0f;
        }
    }
}

// Row strides (elements) of a [batch, heads, rows, D] tensor.
struct Strides {
    int64_t b, h, s;
};

// Keys that some query at positions [first, last] sees, as a stream (see above).
struct KeyStream {
    int a1, delta, length;
};
__device__ __forceinline__ KeyStream key_stream(int first, int last, int keys, int left, int right, int sinks) {
    const int hi = min(last + right, keys - 1);
    const int lo = max(first - left, 0);
    if (hi < 0) return KeyStream{0, 0, 0};
    KeyStream s;
    s.a1 = min(min(sinks, lo), hi + 1);
    s.length = s.a1 + max(hi + 1 - lo, 0);
    s.delta = lo - s.a1;
    return s;
}

}  // namespace peco
