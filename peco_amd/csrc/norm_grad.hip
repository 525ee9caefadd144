// Gradients of the layer norm of norm.hip. With n = (x - m) r of the forward's statistics and g = dy f:
//   dx = r (g - mean(g) - n mean(g n)),  dw = sum over rows of dy n,  db = sum over rows of dy.
// Everything is fp32 but the results, which are rounded once.
//
// HBM-bound: x and dy are read once, dx written once. Each workgroup takes a share of the rows of one entry (of all rows
// where the weight is one for all), keeps its columns' sums of dw and db in registers, joins its wavefronts' sums in LDS
// and writes one row of partial sums of each; a second launch adds those. The shares and the order of every sum depend
// on the sizes alone, so the gradients are the same bits in every call. Measured, both launches: 2 x 7006 x 2048 in bf16 45 us
// (172 MB, 3.8 TB/s; 41 and 4), 24 x 7006 rows of 128 33 us, 2331 x 1111 in fp32 20 us.
#include "rows.hpp"

#include <algorithm>

namespace peco {
namespace {

constexpr int kGradThreads = 512;

struct GradArgs {
    const void *x, *grad, *weight;  // weight nullable: ones
    void* dx;                       // nullable
    const RowStats* stats;
    float* parts;                   // [entries, shares, 2, C], nullable: rows only
    RowMap from, by, to;
    int64_t entry;
    uint32_t entry_rows, shares;
    int channels, waves, wide, around_one;
    float inverse_channels;
};

template <int DT, int L, int kChunks, bool kWhole, bool kSums>
__global__ __launch_bounds__(kGradThreads, kChunks == 1 ? 4 : 2) void norm_grad_kernel(GradArgs a) {
    extern __shared__ float joined[];  // a row of sums
    __shared__ uint32_t slots[2][16];
    constexpr bool kAhead = kChunks < 4 || DT != kF32;  // the next row's loads in flight (as registers allow)
    const int row_lanes = L < kWave ? L : kWave * a.waves;
    const RowLanes r{static_cast<int>(threadIdx.x) % row_lanes, row_lanes, a.channels};
    const uint32_t in_group = row_in_group<L>(row_lanes), group = blockDim.x / row_lanes, step = a.shares * group;
    const uint32_t entry = blockIdx.x / a.shares, share = blockIdx.x - entry * a.shares, before = entry * a.entry_rows;
    RowCombine<L> over{slots, a.waves, static_cast<int>(threadIdx.x / kWave)};
    float w[kChunks][8], dw[kSums ? kChunks : 1][8], db[kSums ? kChunks : 1][8];
    if (a.weight) {
        load_weight<DT, kWhole>(w, a.weight, entry * a.entry, a.wide, r);
        if (a.around_one)
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) w[c][k] += 1.0f;
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) w[c][k] = 1.0f;
    }
    if constexpr (kSums)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) dw[c][k] = db[c][k] = 0.0f;
    Piece<DT> next_x[kChunks], next_g[kChunks];
    RowStats next_stats;
    const auto load = [&](uint32_t in_entry) {
        const uint32_t at = before + min(in_entry, a.entry_rows - 1);
        load_row<DT, kWhole>(next_x, a.x, a.from.at(at), r);
        load_row<DT, kWhole>(next_g, a.grad, a.by.at(at), r);
        next_stats = a.stats[at];
        if (in_entry >= a.entry_rows)  // adds nothing
#pragma unroll
            for (int c = 0; c < kChunks; ++c) next_g[c] = Piece<DT>{};
    };
    uint32_t row = share * group + in_group;
    if (kAhead) load(row);
    for (uint32_t base = share * group; base < a.entry_rows; base += step, row += step) {
        if (!kAhead) load(row);
        Piece<DT> x[kChunks], g[kChunks];
        const RowStats stats = next_stats;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) x[c] = next_x[c], g[c] = next_g[c];
        if (kAhead && base + step < a.entry_rows) load(row + step);
        // n of an element (0 behind the row's end). It is taken from x twice, which costs less than its registers.
        const auto normal = [&](int c, int k) {
            const bool inside = r.template inside<kWhole>(c, k);
            return (x[c].get(k) - (inside ? stats.mean : 0.0f) - (inside ? stats.rest : 0.0f)) * stats.inverse;
        };
        float sum = 0.0f, along = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            __builtin_amdgcn_sched_barrier(0);  // (piece by piece, for the registers)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float n = normal(c, k), d = g[c].get(k), scaled = d * w[c][k];
                if constexpr (kSums) {
                    dw[c][k] = fmaf(d, n, dw[c][k]);
                    db[c][k] += d;
                }
                sum += scaled;
                along = fmaf(scaled, n, along);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) x[c].again(), g[c].again();
        over.sum2(sum, along);
        sum *= a.inverse_channels;
        along *= a.inverse_channels;
        if (row < a.entry_rows && a.dx) {
            const int64_t to = a.to.at(before + row);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                __builtin_amdgcn_sched_barrier(0);
                float dx[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    dx[k] = fmaf(-normal(c, k), along, g[c].get(k) * w[c][k] - sum) * stats.inverse;
                store_piece<DT, kWhole>(round_piece<DT>(dx), a.dx, to, c, r);
            }
        }
    }
    if constexpr (kSums) {
        // The sums of the workgroup's sets of lanes side by side in LDS, then column by column.
        const int sets = L < kWave ? blockDim.x / kWave : group, set = L < kWave ? threadIdx.x / kWave : in_group;
        const int held = row_lanes * kChunks * 8;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&v)[kChunks][8] = which ? db : dw;
            if constexpr (L < kWave) {  // the rows of one wavefront
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int far = L; far < kWave; far *= 2) v[0][k] += wave_shfl_xor(v[0][k], far);
            }
            __syncthreads();
            if (L == kWave || static_cast<int>(threadIdx.x % kWave) < L) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int k = 0; k < 8; ++k) joined[set * held + (c * 8 + k) * row_lanes + r.lane] = v[c][k];
            }
            __syncthreads();
            float* to = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + which) * a.channels;
            for (int e = threadIdx.x; e < held; e += blockDim.x) {
                float sum = joined[e];
                for (int i = 1; i < sets; ++i) sum += joined[i * held + e];
                const int piece = e / row_lanes, lane = e - piece * row_lanes;
                const int col = (piece / 8 * row_lanes + lane) * 8 + piece % 8;
                if (col < a.channels) to[col] = sum;
            }
        }
    }
}

// parts [entries, shares, 2, C] added over the shares: a workgroup takes 64 columns of dw (blockIdx.y 0) or db, its
// wavefronts every 16th share, joined in LDS in order.
constexpr int kJoinWaves = 16;

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __bf16 narrow<__bf16>(float v) { return static_cast<__bf16>(v); }
template <> __device__ __forceinline__ _Float16 narrow<_Float16>(float v) { return static_cast<_Float16>(v); }

template <typename T>
__global__ __launch_bounds__(kWave * kJoinWaves) void join_sums_kernel(const float* parts, T* dweight, T* dbias,
                                                                       uint32_t shares, int channels) {
    __shared__ float sums[kJoinWaves][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int col = blockIdx.x * kWave + lane, which = blockIdx.y;
    T* to = which ? dbias : dweight;
    if (!to) return;
    const int64_t row = 2 * static_cast<int64_t>(channels);
    const float* from = parts + blockIdx.z * shares * row + which * channels + min(col, channels - 1);
    float s[4] = {};
    uint32_t p = wave;
    for (; p + 3 * kJoinWaves < shares; p += 4 * kJoinWaves)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += from[(p + i * kJoinWaves) * row];
    for (; p < shares; p += kJoinWaves) s[0] += from[p * row];
    sums[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (wave || col >= channels) return;
    float total = sums[0][lane];
#pragma unroll
    for (int i = 1; i < kJoinWaves; ++i) total += sums[i][lane];
    to[static_cast<int64_t>(blockIdx.z) * channels + col] = narrow<T>(total);
}

// One piece a lane as long as 8 wavefronts hold the row: two workgroups of 8 wavefronts fit a CU then. Measured over 14012
// rows of 2048 channels in bf16 (with the second launch): 1 piece 39 us, 2 pieces 42, 4 pieces 39; of 1024 channels 25, 26 and
// 29; fp32 rows of 2048 72, 83 and 75.
// Shares of an entry's rows: as many workgroups as fit, fewer where the rows are few.
RowShape grad_shape(int channels) { return row_shape(channels, 1, 8); }
uint32_t grad_shares(const RowShape& s, int entries, uint32_t entry_rows) {
    const int64_t blocks = (s.chunks == 1 ? 2 : 1) * device_compute_units();
    return static_cast<uint32_t>(std::min<int64_t>(std::max<int64_t>(1, blocks / entries), ceil_div(entry_rows, s.rows)));
}

template <int DT, int L, int kChunks, bool kWhole> int launch(const GradArgs& a, const RowShape& s, int entries, hipStream_t st) {
    const dim3 grid(a.shares * entries), block(s.threads);
    if (a.parts) {
        const size_t lds = sizeof(float) * (s.lanes < kWave ? s.threads / kWave : s.rows) * s.lanes * s.waves * kChunks * 8;
        hipLaunchKernelGGL((norm_grad_kernel<DT, L, kChunks, kWhole, true>), grid, block, lds, st, a);
    } else {
        hipLaunchKernelGGL((norm_grad_kernel<DT, L, kChunks, kWhole, false>), grid, block, 0, st, a);
    }
    return hipGetLastError();
}

template <int DT, bool kWhole> int launch_shape(const GradArgs& a, const RowShape& s, int entries, hipStream_t st) {
    if (s.lanes == 8) return launch<DT, 8, 1, kWhole>(a, s, entries, st);
    if (s.lanes == 16) return launch<DT, 16, 1, kWhole>(a, s, entries, st);
    if (s.chunks == 1) return launch<DT, 64, 1, kWhole>(a, s, entries, st);
    if (s.chunks == 2) return launch<DT, 64, 2, kWhole>(a, s, entries, st);
    return launch<DT, 64, 4, kWhole>(a, s, entries, st);
}

template <typename T>
void launch_join(const GradArgs& a, void* dweight, void* dbias, int entries, hipStream_t st) {
    hipLaunchKernelGGL((join_sums_kernel<T>), dim3(static_cast<unsigned>(ceil_div(a.channels, kWave)), 2, entries),
                       dim3(kWave * kJoinWaves), 0, st, a.parts, static_cast<T*>(dweight), static_cast<T*>(dbias),
                       a.shares, a.channels);
}

bool takes(int n0, int n1, int n2, int channels) {
    return n0 >= 1 && n1 >= 1 && n2 >= 1 && channels >= 1 && channels <= kMaxRowChannels &&
           static_cast<int64_t>(n0) * n1 <= 0x3fffffff && static_cast<int64_t>(n0) * n1 * n2 <= 0x3fffffff;
}

}  // namespace
}  // namespace peco

using namespace peco;

PECO_API size_t peco_layer_norm_grad_workspace_size(int n0, int n1, int n2, int channels, int per_entry) {
    if (!takes(n0, n1, n2, channels) || (per_entry && n0 > 65535)) return 0;
    const int entries = per_entry ? n0 : 1;
    const uint32_t rows = static_cast<uint32_t>(n1) * n2 * (per_entry ? 1 : n0);
    return static_cast<size_t>(entries) * grad_shares(grad_shape(channels), entries, rows) * 2 * channels;
}

PECO_API int peco_layer_norm_grad(const void* x, const void* grad, void* dx, const int64_t* strides, const void* weight,
                                  int64_t entry_stride, int wide, int around_one, const float* stats, void* dweight,
                                  void* dbias, int per_entry, float* workspace, size_t workspace_floats, int n0, int n1,
                                  int n2, int channels, int dtype, void* stream) {
    if (!x || !grad || !strides || !stats || entry_stride < 0 || (entry_stride && !per_entry) || n0 < 1 || n1 < 1 ||
        n2 < 1 || channels < 1 || (!dx && !dweight && !dbias))
        return kInvalidValue;
    if (!takes(n0, n1, n2, channels) || (per_entry && n0 > 65535)) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return kUnsupportedDtype;
    const bool sums = dweight || dbias;
    if (sums && (!workspace || workspace_floats < peco_layer_norm_grad_workspace_size(n0, n1, n2, channels, per_entry)))
        return kWorkspaceTooSmall;
    const int entries = per_entry ? n0 : 1;
    GradArgs a{};
    a.x = x;
    a.grad = grad;
    a.weight = weight;
    a.dx = dx;
    a.stats = reinterpret_cast<const RowStats*>(stats);
    a.parts = sums ? workspace : nullptr;
    a.from = row_map(strides, n0, n1, n2);
    a.by = row_map(strides + 3, n0, n1, n2);
    if (dx) a.to = row_map(strides + 6, n0, n1, n2);
    a.entry = entry_stride;
    a.entry_rows = static_cast<uint32_t>(n1) * n2 * (per_entry ? 1 : n0);
    a.channels = channels;
    a.wide = wide;
    a.around_one = around_one;
    a.inverse_channels = 1.0f / static_cast<float>(channels);
    const bool whole = channels % 8 == 0;
    const RowShape s = grad_shape(channels);
    a.shares = grad_shares(s, entries, a.entry_rows);
    a.waves = s.waves;
    const auto st = static_cast<hipStream_t>(stream);
    int status;
    switch (dtype) {
        case kBF16: status = whole ? launch_shape<kBF16, true>(a, s, entries, st) : launch_shape<kBF16, false>(a, s, entries, st); break;
        case kF16: status = whole ? launch_shape<kF16, true>(a, s, entries, st) : launch_shape<kF16, false>(a, s, entries, st); break;
        default: status = whole ? launch_shape<kF32, true>(a, s, entries, st) : launch_shape<kF32, false>(a, s, entries, st);
    }
    if (status || !sums) return status;
    if (wide || dtype == kF32) launch_join<float>(a, dweight, dbias, entries, st);
    else if (dtype == kBF16) launch_join<__bf16>(a, dweight, dbias, entries, st);
    else launch_join<_Float16>(a, dweight, dbias, entries, st);
    return hipGetLastError();
}
