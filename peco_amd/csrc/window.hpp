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

#include <algorithm>

namespace peco {

constexpr int kWinTile = 64;      // rows of an LDS tile
constexpr int kWinRows = 128;     // query rows of a forward or dQ workgroup, keys of a dK/dV workgroup
constexpr int kUnbounded = 0x40000000;  // left or right without a limit

// Scaled scores past which the reference is subtracted before the multiplication: exp2(fma(s, scale, -m scale))
// rounds m * scale first, 2^-14 of an exponent off at this size.
constexpr float kWideScores = 0x1p10f;

template <int D> struct WinTile {
    static constexpr int CH = D / 8;                 // 16-byte chunks per row
    static constexpr int kElems = kWinTile * D;
    static constexpr int kWaveRows = kWave / CH;     // rows per wave-wide direct load
    static constexpr int kLoads = kWinTile / (4 * kWaveRows);  // direct loads per wave per tile (4 waves)
    static __device__ __forceinline__ int swz(int row) {
        return CH == 16 ? 4 * (row % 4) + ((row >> 2) & 3) : 4 * ((row >> 1) & 1) + ((row >> 2) & 3);
    }
};

// LDS addresses (bytes) of a lane's fragments of the tile at address 0 of the workgroup's tiles. The steps of a row
// of fragments differ from one another in bits of the swizzled chunk alone, so one address each and exclusive ors
// give all of them; a tile's and a half's distance from the first tile are constants that go into the LDS reads'
// immediate offsets. The tiles start on a multiple of 256 bytes.
typedef __attribute__((address_space(3))) const u16x8* LdsChunk;
template <int D> struct WinLane {
    int row;      // A operand with rows along M: row l % 32, channels 8 (l / 32) .. + 7
    int channel;  // A operand with channels along M: see channels()
    __device__ __forceinline__ WinLane(int lane, const uint16_t* tiles) {
        using T = WinTile<D>;
        const int h = lane / 32, r = lane % 32, src = lane % 16, at = 4 * h + src / 4;
        const int base = static_cast<int>(lds_addr(tiles));
        row = base + 2 * (r * D + (h ^ T::swz(r)) * 8);
        const int d = 16 * ((lane / 16) % 2) + 4 * (src % 4);
        channel = base + 2 * (at * D + ((d / 8) ^ T::swz(at)) * 8 + d % 8);
    }
    // The same `bytes` (a multiple of 256) further on.
    __device__ __forceinline__ WinLane moved(int bytes) const {
        WinLane x = *this;
        x.row += bytes;
        x.channel += bytes;
        return x;
    }
    // Keeps the compiler from computing every address once and holding them all through a loop.
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(row), "+v"(channel)); }
    // The 32 rows at byte `off` (a multiple of 16 rows: the swizzle repeats every 16), channels 16 s + 8 (l / 32) ...
    __device__ __forceinline__ u16x8 rows(int off, int s) const { return *LdsChunk((row ^ (32 * s)) + off); }
    // Channel 32 nb + l % 32 of rows 8 u + 4 (l / 32) + (0..3), u = 0, 1, from byte `off` on (a multiple of 16 rows),
    // by transpose reads: source lane r of each 16-lane group points at row r / 4, channels 32 nb + 16 ((l / 16) % 2)
    // + 4 (r % 4).
    __device__ __forceinline__ u16x8 channels(int off, int nb) const {
        u32x2 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            part[u] = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                           (channel ^ (64 * nb + 32 * u)) + (off + 16 * u * D))));
        return __builtin_bit_cast(u16x8, u32x4{part[0][0], part[0][1], part[1][0], part[1][1]});
    }
};

template <int DT> __device__ __forceinline__ bool not_finite(uint16_t b) {
    constexpr uint16_t kExp = DT == kBF16 ? 0x7f80 : 0x7c00;
    return (b & kExp) == kExp;
}

template <int N> __device__ __forceinline__ bool all_finite(const f32x16 (&acc)[N]) {
    float zero = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(acc[n][i], 0.0f, zero);
    return zero == 0.0f;
}

// Whether any of the 32 rows at byte `off` of the tiles holds an infinity or NaN.
template <int DT, int D>
__device__ __forceinline__ bool rows_not_finite(const uint16_t* tiles, int off, int lane) {
    bool bad = false;
#pragma unroll 1
    for (int i = 0; i < 32 * D / 8 / kWave; ++i) {
        const u16x8 x = *reinterpret_cast<const u16x8*>(tiles + off / 2 + (i * kWave + lane) * 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) bad |= not_finite<DT>(x[k]);
    }
    return __any(bad);
}

// Schedules the kProducts products before it with the kReads LDS reads of their operands, kAhead of them before the
// first product and the others spread over the products (LDS latency is longer than a product; more in flight costs
// registers).
template <int kProducts, int kReads, int kAhead> __device__ __forceinline__ void read_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);  // LDS reads
    constexpr int kRest = kReads - kAhead, kEach = (kRest + kProducts - 1) / kProducts;
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        if (i * kEach < kRest) __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
    }
}

// acc += (the 32 rows at byte `off`, channels along M) x w, where w holds this lane's column: packed weight pairs of
// rows 8 (i / 4) + 4 h + i % 4.
template <int DT, int D>
__device__ __forceinline__ void add_rows(f32x16 (&acc)[D / 32], int off, const uint32_t (&w)[8],
                                         const WinLane<D>& at) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const u16x8 b = __builtin_bit_cast(u16x8, u32x4{w[4 * kk], w[4 * kk + 1], w[4 * kk + 2], w[4 * kk + 3]});
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
            acc[nb] = Mfma<DT>::run(at.channels(off + 32 * kk * D, nb), b, acc[nb]);
    }
    read_ahead<D / 16, D / 8, 6>();
}

// The same for rows with infinities or NaN that some column hides: a hidden row's weight is 0, but 0 times them is
// NaN. The products take such elements as 0, in add_rows' order, so that columns that hide them come out bit for bit as
// without them; then the elements of one row after another are multiplied by themselves and added where seen(row) holds.
// The kernels come here only in a second walk over their tiles, after the sums of a first one came out other than finite.
template <int DT, int D, typename Seen>
__device__ __forceinline__ void add_rows_seen(f32x16 (&acc)[D / 32], int off, const uint32_t (&w)[8],
                                              const WinLane<D>& at, int h, const Seen& seen) {
    auto weights = [&](int kk) {
        return __builtin_bit_cast(u16x8, u32x4{w[4 * kk], w[4 * kk + 1], w[4 * kk + 2], w[4 * kk + 3]});
    };
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb) {
            u16x8 a = at.channels(off + 32 * kk * D, nb);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (not_finite<DT>(a[e])) a[e] = 0;
            acc[nb] = Mfma<DT>::run(a, weights(kk), acc[nb]);
            __builtin_amdgcn_sched_barrier(0);  // (one operand at a time: the sums leave few registers)
        }
#pragma unroll 1
    for (int row = 0; row < 32; ++row) {
        const bool add = seen(row);
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u16x8 a = at.channels(off + 32 * kk * D, nb);
                bool any = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool take = 16 * kk + 8 * (e / 4) + 4 * h + e % 4 == row && not_finite<DT>(a[e]);
                    if (!take) a[e] = 0;
                    any |= take;
                }
                if (!__any(any)) continue;
                const f32x16 one = Mfma<DT>::run(a, weights(kk), f32x16{});
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

// Most keys that a tile of `tokens` tokens' rows may see.
inline int64_t seen_keys(int64_t keys, int64_t tokens, int left, int right, int sinks) {
    const int64_t window = left < 0 || right < 0 ? keys : std::min<int64_t>(keys, int64_t{left} + right + tokens + sinks);
    return std::max<int64_t>(window, 0);
}

constexpr int kPartTiles = 4;   // of a part at least
constexpr int kStartTiles = 4;
constexpr int kMaxSplits = 64;
inline int64_t most_parts(int64_t keys) {
    return std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, ceil_div(keys, kWinTile) / kPartTiles));
}

// Into how many parts the walks of `items` row tiles, each over up to `keys` keys, `rows` query rows in all, are cut.
// A call takes as long as its busiest CU: the count of workgroups there times a workgroup's tiles (and kStartTiles for
// its start and end), in units of what a CU takes for a tile with two workgroups sharing it (1.3 to 1.4 us with 128
// channels, half with 64, in the forward and in dQ; one alone is a third faster than that, not twice), plus the join, which
// writes and reads the parts' fp32 rows.
inline int cut_parts(int64_t items, int64_t keys, int64_t rows, int d) {
    const int64_t cus = device_compute_units(), n = ceil_div(keys, kWinTile), most = most_parts(keys);
    const double tile_us = d == 128 ? 1.4 : 0.7;
    double least = 1e30;
    int best = 1;
    for (int s = 1; s <= most; ++s) {
        const int64_t k = ceil_div(items * s, cus);
        double cost = (k == 1 ? 4.0 / 3.0 : static_cast<double>(k)) * static_cast<double>(ceil_div(n, s) + kStartTiles);
        if (s > 1) cost += (4.0 + static_cast<double>(rows) * s * (d + 2) * 8.0 / 5.0e6) / tile_us;  // 4 us and 5 TB/s
        else cost *= 0.93;  // (less than that a cut is not worth: the busiest CU's last workgroup runs the faster)
        if (cost >= least) continue;
        least = cost;
        best = s;
    }
    return best;
}

}  // namespace peco
