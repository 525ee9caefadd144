// Layer norm over a row's channels, rows quantized to 8 bits, and both at once.
//
// Norm: m = sum x / C, v = sum (x - m)^2 / C, r = 1 / sqrt(v + eps), y = (x - m) r f + b with f = w or 1 + w, all in fp32
// and rounded once to the rows' type. The row is in registers, so its deviations are taken from the mean itself (the
// difference of E[x^2] and m^2 would cancel for rows far from 0), and the mean is kept in two parts: what rounding left of
// it is the mean of those deviations. An error of half a step of the mean would stay in every deviation, which for
// rows much further from 0 than they are wide is no small part of them. w and b are one row for all, or one for each entry of
// the outermost axis (a modulation).
//
// Quantized rows: a = max |x|, code = rint(x * (127 * (1 / a))), scale = a * (1 / 127), each operation in fp32 (IEEE), halves
// to even. For 16-bit rows these are the codes nearest to the real quotients: x * 127 / a is 2^-20 or more off any half
// that it does not meet exactly, and the three roundings move it by 2^-22 of itself; where it is a half (x = a / 2), both
// neighbours are. A row whose largest magnitude is below 127 * 2^-126, where the scale would leave the normal numbers,
// counts as 0 (codes and scale 0). A row with an infinity or a NaN gets codes 0 and a NaN as its scale, which makes its
// products NaN and no others. The norm's rows are quantized from their fp32 values.
//
// HBM-bound: a row is read once and its result written once. Workgroups walk over rows with the next row's loads in flight
// while one is normalised, and keep the weight in registers for all of their rows. Measured: norm of 119056 x 4096 in fp16
// 336-348 us (1.95 GB, 5.7 TB/s; a copy of 1 GB runs at 5.05-5.08), 7006 x 2048 in bf16 12-13 us (4.6), 24 x 7006 rows of 128
// with their statistics 16-20 us; codes of 119056 x 4096 247 us (1.46 GB, 5.9), of 7006 x 2048 8-10 us, of its norm 12-14 us.
#include "rows.hpp"

#include <algorithm>
#include <atomic>

namespace peco {
namespace {

enum Mode { kNorm, kNormCodes, kCodes };

struct NormArgs {
    const void* x;
    const void *weight, *bias;  // nullable
    void* out;                  // kNorm
    RowStats* stats;            // kNorm, nullable
    int8_t* codes;              // the others
    float* scales;
    RowMap from, to;
    int64_t pitch;              // bytes between rows of codes
    int64_t entry;              // elements between the weights of two entries, 0: one for all
    uint32_t rows, entry_rows;
    int channels, waves, wide, around_one;
    float eps, inverse_channels;
};

template <int DT, int L, int kChunks, bool kWhole, int kMode>
__global__ __launch_bounds__(512) void norm_kernel(NormArgs a) {
    __shared__ uint32_t slots[2][16];
    const int row_lanes = L < kWave ? L : kWave * a.waves;
    const RowLanes r{static_cast<int>(threadIdx.x) % row_lanes, row_lanes, a.channels};
    const uint32_t in_group = row_in_group<L>(row_lanes), group = blockDim.x / row_lanes, step = gridDim.x * group;
    RowCombine<L> over{slots, a.waves, static_cast<int>(threadIdx.x / kWave)};
    float w[kChunks][8], b[kChunks][8];
    uint32_t held = ~0u;  // the entry that w and b are of
    if constexpr (kMode != kCodes) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[c][k] = 1.0f, b[c][k] = 0.0f;
    }
    Piece<DT> next[kChunks];
    uint32_t row = blockIdx.x * group + in_group;  // (the workgroup's rows stay together: its barriers are met by all)
    load_row<DT, kWhole>(next, a.x, a.from.at(min(row, a.rows - 1)), r);
    for (uint32_t base = blockIdx.x * group; base < a.rows; base += step, row += step) {
        const uint32_t at = min(row, a.rows - 1);
        float x[kChunks][8];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) x[c][k] = next[c].get(k);
        if (base + step < a.rows)
            load_row<DT, kWhole>(next, a.x, a.from.at(min(row + step, a.rows - 1)), r);
        if constexpr (kMode != kCodes) {
            const uint32_t entry = a.entry ? at / a.entry_rows : 0;
            if (entry != held && (a.weight || a.bias)) {
                held = entry;
                if (a.weight) load_weight<DT, kWhole>(w, a.weight, entry * a.entry, a.wide, r);
                if (a.bias) load_weight<DT, kWhole>(b, a.bias, entry * a.entry, a.wide, r);
                if (a.around_one)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[c][k] += 1.0f;
            }
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += x[c][k];
            const float mean = over.sum(sum) * a.inverse_channels;
            float rest = 0.0f, squares = 0.0f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[c][k] -= r.template inside<kWhole>(c, k) ? mean : 0.0f;  // (0 behind the row's end)
                    rest += x[c][k];
                    squares = fmaf(x[c][k], x[c][k], squares);
                }
            over.sum2(rest, squares);
            rest *= a.inverse_channels;
            const float variance = squares * a.inverse_channels - rest * rest;
            const float inverse = 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + a.eps);
            if (kMode == kNorm && a.stats && r.lane == 0 && row < a.rows) a.stats[row] = RowStats{mean, rest, inverse};
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[c][k] -= r.template inside<kWhole>(c, k) ? rest : 0.0f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[c][k] = fmaf(x[c][k] * inverse, w[c][k], b[c][k]);
        }
        if constexpr (kMode == kNorm) {
            if (row < a.rows) {
                const int64_t to = a.to.at(row);
#pragma unroll
                for (int c = 0; c < kChunks; ++c) store_piece<DT, kWhole>(round_piece<DT>(x[c]), a.out, to, c, r);
            }
        } else {
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(x[c][k]) & 0x7fffffffu);
            most = over.template run<MaxU>(most);
            const RowScale scale(most);
            if (row < a.rows) {
                if (r.lane == 0) a.scales[row] = scale.scale();
                int8_t* to = a.codes + row * a.pitch;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    int code[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) code[k] = scale.code(x[c][k]);
                    u32x2 packed{};
#pragma unroll
                    for (int k = 0; k < 8; ++k) packed[k / 4] |= (code[k] & 0xffu) << (8 * (k % 4));
                    const int col = r.first(c);
                    if (col < a.channels) *reinterpret_cast<u32x2*>(to + col) = packed;
                }
            }
        }
    }
}

// Workgroups of this kind that a CU holds at once (all devices are alike; asked once for each size of a workgroup).
template <int DT, int L, int kChunks, bool kWhole, int kMode> int resident(int threads) {
    static std::atomic<int> known[512 / kWave + 1];
    int n = known[threads / kWave].load(std::memory_order_relaxed);
    if (!n) {
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_kernel<DT, L, kChunks, kWhole, kMode>, threads, 0) != hipSuccess || n < 1)
            n = 1;
        known[threads / kWave].store(n, std::memory_order_relaxed);
    }
    return n;
}

// As many workgroups as fit: each then walks over several rows with the next one's loads in flight, and keeps its weight. Of
// 8 a CU, where 3 fit, most had one row: 7006 x 2048 in bf16 14.6 us for 12.5, 2 x 7006 with statistics 25.9 for 21.9.
template <int DT, int L, int kChunks, bool kWhole, int kMode>
int launch(const NormArgs& a, const RowShape& s, hipStream_t stream) {
    int groups = resident<DT, L, kChunks, kWhole, kMode>(s.threads);
    if (kMode == kCodes && kWhole) {
        // Codes alone are quickest with 3 a CU (300000 x 1024 in bf16 165 us, with 4 or 8 176 and 181), rows of 4 pieces that
        // do not stay in the 256 MB of the last cache with 2 (119056 x 4096 247 us, 272 with 3; 7006 x 4096 16.8 and 15.7).
        const int64_t bytes = static_cast<int64_t>(a.rows) * a.channels * (DT == kF32 ? 4 : 2);
        groups = std::min(groups, kChunks == 4 && bytes > int64_t{256} << 20 ? 2 : 3);
    }
    const int64_t blocks = std::min<int64_t>(ceil_div(a.rows, s.rows), static_cast<int64_t>(groups) * device_compute_units());
    hipLaunchKernelGGL((norm_kernel<DT, L, kChunks, kWhole, kMode>), dim3(static_cast<unsigned>(blocks)),
                       dim3(s.threads), 0, stream, a);
    return hipGetLastError();
}

template <int DT, bool kWhole, int kMode> int launch_shape(const NormArgs& a, const RowShape& s, hipStream_t stream) {
    if (s.lanes == 8) return launch<DT, 8, 1, kWhole, kMode>(a, s, stream);
    if (s.lanes == 16) return launch<DT, 16, 1, kWhole, kMode>(a, s, stream);
    if (s.chunks == 1) return launch<DT, 64, 1, kWhole, kMode>(a, s, stream);
    if (s.chunks == 2) return launch<DT, 64, 2, kWhole, kMode>(a, s, stream);
    return launch<DT, 64, 4, kWhole, kMode>(a, s, stream);
}

// Pieces a lane: up to 4 of 16 bytes keep a row of 2048 channels in one wavefront, whose sums need no barrier (119056 x 4096
// in fp16: 349 us with 4 pieces, 395 with 2; 2048 x 2048 in bf16 5.1, 5.9 and, with 1, 7.1). Two where a piece is 32 bytes or
// rows end inside a piece, whose moves take registers (7006 x 2048 in fp32 25.2, 22.9 and 21.7, 7006 x 4096 41.4, 36.8 and 39.5;
// 7006 x 2047 in bf16 21.5, 16.2 and 18.2).
template <int kMode> int launch_type(NormArgs a, int dtype, hipStream_t stream) {
    const bool whole = a.channels % 8 == 0;
    const RowShape s = row_shape(a.channels, whole && dtype != kF32 ? 4 : 2, 4);
    a.waves = s.waves;
    switch (dtype) {
        case kBF16: return whole ? launch_shape<kBF16, true, kMode>(a, s, stream) : launch_shape<kBF16, false, kMode>(a, s, stream);
        case kF16: return whole ? launch_shape<kF16, true, kMode>(a, s, stream) : launch_shape<kF16, false, kMode>(a, s, stream);
        default: return whole ? launch_shape<kF32, true, kMode>(a, s, stream) : launch_shape<kF32, false, kMode>(a, s, stream);
    }
}

// Sizes that every entry takes: kOk, or why not.
int check_rows(const void* x, const int64_t* strides, int n0, int n1, int n2, int channels, int dtype) {
    if (!x || !strides || n0 < 1 || n1 < 1 || n2 < 1 || channels < 1) return kInvalidValue;
    if (channels > kMaxRowChannels || static_cast<int64_t>(n0) * n1 > 0x3fffffff ||
        static_cast<int64_t>(n0) * n1 * n2 > 0x3fffffff)
        return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return kUnsupportedDtype;
    return kOk;
}

void set_rows(NormArgs& a, const void* x, const int64_t* strides, int n0, int n1, int n2, int channels) {
    a.x = x;
    a.from = row_map(strides, n0, n1, n2);
    a.rows = static_cast<uint32_t>(n0) * n1 * n2;
    a.entry_rows = static_cast<uint32_t>(n1) * n2;
    a.channels = channels;
    a.inverse_channels = 1.0f / static_cast<float>(channels);
}

void set_affine(NormArgs& a, const void* weight, const void* bias, int64_t entry, int wide, int around_one, float eps) {
    a.weight = weight;
    a.bias = bias;
    a.entry = entry;
    a.wide = wide;
    a.around_one = around_one && weight;
    a.eps = eps;
}

}  // namespace

int launch_quantize_rows(const void* x, const int64_t* strides, int8_t* codes, int64_t pitch, float* scales, int n0,
                         int n1, int n2, int channels, int dtype, hipStream_t stream) {
    if (const int bad = check_rows(x, strides, n0, n1, n2, channels, dtype)) return bad;
    if (!codes || !scales || pitch < channels || pitch % 16 || reinterpret_cast<uintptr_t>(codes) % 16) return kInvalidValue;
    NormArgs a{};
    set_rows(a, x, strides, n0, n1, n2, channels);
    a.codes = codes;
    a.scales = scales;
    a.pitch = pitch;
    return launch_type<kCodes>(a, dtype, stream);
}

}  // namespace peco

using namespace peco;

PECO_API int peco_layer_norm(const void* x, void* output, const int64_t* strides, const void* weight, const void* bias,
                             int64_t entry_stride, int wide, int around_one, float eps, float* stats, int n0, int n1,
                             int n2, int channels, int dtype, void* stream) {
    if (const int bad = check_rows(x, strides, n0, n1, n2, channels, dtype)) return bad;
    if (!output || entry_stride < 0) return kInvalidValue;
    NormArgs a{};
    set_rows(a, x, strides, n0, n1, n2, channels);
    set_affine(a, weight, bias, entry_stride, wide, around_one, eps);
    a.out = output;
    a.to = row_map(strides + 3, n0, n1, n2);
    a.stats = reinterpret_cast<RowStats*>(stats);
    return launch_type<kNorm>(a, dtype, static_cast<hipStream_t>(stream));
}

PECO_API int peco_layer_norm_rows(const void* x, const int64_t* strides, const void* weight, const void* bias,
                                  int64_t entry_stride, int wide, int around_one, float eps, int8_t* codes,
                                  int64_t pitch, float* scales, int n0, int n1, int n2, int channels, int dtype,
                                  void* stream) {
    if (const int bad = check_rows(x, strides, n0, n1, n2, channels, dtype)) return bad;
    if (!codes || !scales || entry_stride < 0 || pitch < channels || pitch % 16 || reinterpret_cast<uintptr_t>(codes) % 16)
        return kInvalidValue;
    NormArgs a{};
    set_rows(a, x, strides, n0, n1, n2, channels);
    set_affine(a, weight, bias, entry_stride, wide, around_one, eps);
    a.codes = codes;
    a.scales = scales;
    a.pitch = pitch;
    return launch_type<kNormCodes>(a, dtype, static_cast<hipStream_t>(stream));
}

PECO_API int peco_quantize_rows(const void* x, const int64_t* strides, int8_t* codes, int64_t pitch, float* scales,
                                int n0, int n1, int n2, int channels, int dtype, void* stream) {
    return launch_quantize_rows(x, strides, codes, pitch, scales, n0, n1, n2, channels, dtype,
                                static_cast<hipStream_t>(stream));
}
