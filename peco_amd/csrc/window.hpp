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
};

// Where a lane's fragments lie in a tile (bytes from its first row). Kept apart from the tile and the row block,
// which are constants of the unrolled loops and go into the LDS reads' immediate offsets.
template <int D> struct WinLane {
    using T = WinTile<D>;
    int row[D / 16];        // A operand with rows along M: row l % 32, channels 16 s + 8 (l / 32) .. + 7
    int channel[D / 32][2]; // A operand with channels along M (see channels below)
    __device__ __forceinline__ explicit WinLane(int lane) {
        const int h = lane / 32, r = lane % 32;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) row[s] = 2 * (r * D + ((2 * s + h) ^ T::swz(r)) * 8);
        const int src = lane % 16;
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 32 * nb + 16 * ((lane / 16) % 2) + 4 * (src % 4), at = 8 * u + 4 * h + src / 4;
                channel[nb][u] = 2 * (at * D + ((d / 8) ^ T::swz(at)) * 8 + d % 8);
            }
    }
    // Rows row0 .. row0 + 31 (row0 a multiple of 32; the swizzle repeats every 16 rows), step s.
    __device__ __forceinline__ u16x8 rows(const uint16_t* t, int row0, int s) const {
        return *reinterpret_cast<const u16x8*>(reinterpret_cast<const char*>(t) + (row[s] + 2 * row0 * D));
    }
    // Channel 32 nb + l % 32 of tile rows row0 + 8 u + 4 (l / 32) + (0..3), u = 0, 1 (row0 a multiple of 16), by
    // transpose reads: source lane r of each 16-lane group points at row r / 4, channels 32 nb + 16 ((l / 16) % 2) +
    // 4 (r % 4).
    __device__ __forceinline__ u16x8 channels(const uint16_t* t, int row0, int nb) const {
        u32x2 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* a = reinterpret_cast<const char*>(t) + (channel[nb][u] + 2 * row0 * D);
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
#pragma unroll 1
    for (int i = 0; i < 32 * D / 8 / kWave; ++i) {
        const u16x8 x = *reinterpret_cast<const u16x8*>(t + row0 * D + (i * kWave + lane) * 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) bad |= not_finite<DT>(x[k]);
    }
    return __any(bad);
}

// Schedules the N products before it with their A fragments, one LDS read each, read four products ahead (LDS
// latency is longer than a product; more in flight costs registers).
template <int N> __device__ __forceinline__ void read_ahead() {
    constexpr int kAhead = 4;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

// The same for N products whose A fragments are two transpose reads each.
template <int N> __device__ __forceinline__ void read_channels_ahead() {
    constexpr int kAhead = 3;
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

// acc += (tile rows row0 .. row0 + 31, channels along M) x w, where w holds this lane's column: packed weight
// pairs of rows 8 (i / 4) + 4 h + i % 4.
template <int DT, int D>
__device__ __forceinline__ void add_rows(f32x16 (&acc)[D / 32], const uint16_t* t, int row0, const uint32_t (&w)[8],
                                         const WinLane<D>& at) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const u16x8 b = __builtin_bit_cast(u16x8, u32x4{w[4 * kk], w[4 * kk + 1], w[4 * kk + 2], w[4 * kk + 3]});
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
            acc[nb] = Mfma<DT>::run(at.channels(t, row0 + 16 * kk, nb), b, acc[nb]);
    }
    read_channels_ahead<D / 16>();
}

// The same for a tile with infinities or NaN in rows that some column hides: a hidden row's weight is 0, but 0
// times them is NaN. Each tile row is multiplied by itself and added where seen(row) holds. The kernels come
// here only in a second walk over their tiles, after a first one met such a tile.
template <int DT, int D, typename Seen>
__device__ __forceinline__ void add_rows_seen(f32x16 (&acc)[D / 32], const uint16_t* t, int row0,
                                              const uint32_t (&w)[8], const WinLane<D>& at, int h, const Seen& seen) {
#pragma unroll 1
    for (int row = 0; row < 32; ++row) {
        const bool add = seen(row);
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb) {
            f32x16 one{};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u16x8 a = at.channels(t, row0 + 16 * kk, nb);
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

// 16 bytes a lane of row `row` (`stride` elements apart) of a head, at byte `chunk`, into LDS. kFar: the head's
// rows span more than 2^32 bytes.
template <bool kFar>
__device__ __forceinline__ void load_row16(const uint16_t* head, int row, int64_t stride, uint32_t chunk, uint32_t lds) {
    if constexpr (kFar) dma16(head + row * stride + chunk / 2, lds);
    else dma16_off(head, static_cast<uint32_t>(row) * static_cast<uint32_t>(2 * stride) + chunk, lds);
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
