// Rotary positions with several axes over strided rows, forward and (with the inverse rotation) backward.
//
// x [batch, heads, rows, D] (any strides, channels adjacent, rows on 16 bytes) to an output of the same
// shape and its own strides. The first 2 P channels of a row form P pairs, adjacent channels (2 i, 2 i + 1)
// or halves (i, i + P), and pair i turns by its axis's position times its frequency (rotary.hpp):
//   (a, b) -> (a cos - b sin, b cos + a sin), in fp32, rounded once to the type.
// The rotation is orthogonal, so the gradient of the rows is the gradient of the output turned back.
//
// HBM-bound: each row is read and written once and the angles are computed, so no tables are read (fp32
// tables of 118800 rows x 128 channels are 122 MB, a sixth of what 24 bf16 heads move, for each group of
// heads that reads them). A lane holds 8 channels (16 for halves: 8 of each) of one row of kHeads heads with
// all loads in flight and computes its 4 (8) angles once for all of them. Measured, 24 heads x 128 channels, bf16:
// 6750 rows 18 us (83 MB, 4.6 TB/s; a plain copy reaches 5.2), 118800 rows in halves 317 us (1.46 GB, 4.6 TB/s).
#include "rotary.hpp"

namespace peco {
namespace {

struct RotaryArgs {
    const void* in;
    void* out;
    int64_t in_batch, in_head, in_row;  // strides in elements
    int64_t out_batch, out_head, out_row;
    int batch, heads, dims;
    uint32_t rows;
    uint32_t lanes;  // lanes per row
};

template <int DT, bool kHalves, int kHeads>
__global__ __launch_bounds__(256) void rotary_axes_kernel(RotaryArgs a, RotaryPlan plan) {
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    const uint32_t row = item / a.lanes;
    if (row >= a.rows) return;
    const int lane = static_cast<int>(item - row * a.lanes);
    const int h0 = blockIdx.y * kHeads;
    constexpr int kChunks = kHalves ? 2 : 1;
    constexpr int kPairs = kHalves ? 8 : 4;
    // Channels of this lane's chunks. Halves: chunk `lane` of either half, then one chunk a lane behind them.
    const int half_lanes = plan.pairs / 8;
    const bool tail = kHalves ? lane >= half_lanes : 4 * lane >= plan.pairs;
    const int c0 = kHalves && tail ? 8 * (lane + half_lanes) : 8 * lane;
    const int c1 = kHalves && !tail ? plan.pairs + 8 * lane : c0;
    for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
        const int64_t src = b * a.in_batch + static_cast<int64_t>(row) * a.in_row;
        const int64_t dst = b * a.out_batch + static_cast<int64_t>(row) * a.out_row;
        Chunk<DT> x[kHeads][kChunks];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {  // clamped, unconditional: all loads in flight
            const int64_t at = src + static_cast<int64_t>(min(h0 + i, a.heads - 1)) * a.in_head;
            x[i][0].load(a.in, at + c0);
            if constexpr (kHalves) x[i][1].load(a.in, at + c1);
        }
        if (!tail) {
            float c[kPairs], s[kPairs];
            rotary_angles<kPairs>(plan, b, row, kPairs * lane, c, s);
#pragma unroll
            for (int i = 0; i < kHeads; ++i) {
                if constexpr (kHalves) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float u = x[i][0].get(k), v = x[i][1].get(k);
                        x[i][0].set(k, u * c[k] - v * s[k]);
                        x[i][1].set(k, v * c[k] + u * s[k]);
                    }
                } else {
                    turn_adjacent(x[i][0], 4 * lane, plan.pairs, c, s);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (h0 + i >= a.heads) break;
            const int64_t at = dst + static_cast<int64_t>(h0 + i) * a.out_head;
            x[i][0].store(a.out, at + c0);
            if constexpr (kHalves) {
                if (!tail) x[i][1].store(a.out, at + c1);
            }
        }
    }
}

// Heads per lane: 8 keep 128 bytes a lane in flight for 16-bit rows; the wider forms take 4 for the registers.
template <int DT, bool kHalves> int launch_rotary(const RotaryArgs& a, const RotaryPlan& plan, hipStream_t s) {
    constexpr int kHeads = DT == kF32 || kHalves ? 4 : 8;
    const int64_t blocks = ceil_div(static_cast<int64_t>(a.rows) * a.lanes, 256);
    const int64_t groups = ceil_div(a.heads, kHeads);
    if (groups > 65535) return kUnsupportedShape;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups),
                    static_cast<unsigned>(a.batch < 65535 ? a.batch : 65535));
    hipLaunchKernelGGL((rotary_axes_kernel<DT, kHalves, kHeads>), grid, dim3(256), 0, s, a, plan);
    return hipGetLastError();
}

// New tokens' keys (rotated) and values into the pages of a cache. k and v [tokens, heads, D] hold the tokens of
// `batch` sequences in a row (offsets), token i of n of sequence b goes to place lengths[b] - n + i of its row of
// the page table. Every lane moves 8 channels of K and of V of kHeads heads of one token; with halves it reads
// its partner chunk as well (from the L1, where the partner's own read puts it). Measured, 128 channels, bf16: 5497
// tokens of 24 heads 29 us (135 MB, 4.7 TB/s), 32 tokens of 8 heads 6 us.
struct AppendArgs {
    const uint16_t *k, *v;
    uint16_t *k_pages, *v_pages;
    int64_t k_token, k_head, v_token, v_head;         // strides in elements
    int64_t kp_page, kp_head, kp_row, vp_page, vp_head, vp_row;
    const int32_t *table, *offsets, *lengths;
    int64_t table_stride;
    int batch, heads, tokens, pages, page, width;
    int halves;
};

template <int DT, int D, int kHeads>
__global__ __launch_bounds__(256) void append_pages_kernel(AppendArgs a, RotaryPlan plan) {
    constexpr int G = D / 8;               // lanes a token
    constexpr int kTokens = kWave / G;     // tokens a wavefront
    const int lane = threadIdx.x % kWave;
    const int first = (blockIdx.x * (256 / kWave) + threadIdx.x / kWave) * kTokens;
    if (first >= a.tokens) return;
    const int token = first + lane / G;
    // The token's sequence: the offsets up to it, counted 64 at a time for all the wavefront's tokens.
    int upto = 0;
    for (int b0 = 0; b0 <= a.batch; b0 += kWave) {
        const int at = b0 + lane;
        const int offset = at <= a.batch ? a.offsets[at] : 0x7fffffff;
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            const int n = __popcll(__ballot(offset <= first + t));
            upto += lane / G == t ? n : 0;
        }
    }
    const int b = upto - 1;
    if (token >= a.tokens || b < 0 || b >= a.batch) return;  // of no sequence
    const int begin = max(0, a.offsets[b]), end = min(a.offsets[b + 1], a.tokens);
    const int64_t place = static_cast<int64_t>(a.lengths[b]) - (end - begin) + (token - begin);
    if (place < 0 || place >= static_cast<int64_t>(a.width) * a.page) return;
    const int page = a.table[b * a.table_stride + place / a.page];
    if (page < 0 || page >= a.pages) return;  // not held
    const int64_t slot = place % a.page;
    const int c = 8 * (lane % G), chunk = lane % G, h0 = blockIdx.y * kHeads;
    const int half = plan.pairs / 8;  // chunks of a half
    const bool turns = a.halves ? chunk < 2 * half : c < 2 * plan.pairs;
    const int partner = a.halves && turns ? (chunk < half ? c + plan.pairs : c - plan.pairs) : c;
    Chunk<DT> kx[kHeads], px[kHeads], vx[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int head = min(h0 + i, a.heads - 1);
        kx[i].load(a.k, token * a.k_token + head * a.k_head + c);
        if (a.halves) px[i].load(a.k, token * a.k_token + head * a.k_head + partner);
        vx[i].load(a.v, token * a.v_token + head * a.v_head + c);
    }
    if (turns) {
        if (a.halves) {
            const bool upper = chunk >= half;
            float cs[8], sn[8];
            rotary_angles<8>(plan, 0, token, 8 * (upper ? chunk - half : chunk), cs, sn);
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float own = kx[i].get(k), other = px[i].get(k);
                    kx[i].set(k, upper ? own * cs[k] + other * sn[k] : own * cs[k] - other * sn[k]);
                }
        } else {
            float cs[4], sn[4];
            rotary_angles<4>(plan, 0, token, c / 2, cs, sn);
#pragma unroll
            for (int i = 0; i < kHeads; ++i) turn_adjacent(kx[i], c / 2, plan.pairs, cs, sn);
        }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        if (h0 + i >= a.heads) break;
        kx[i].store(a.k_pages, page * a.kp_page + (h0 + i) * a.kp_head + slot * a.kp_row + c);
        vx[i].store(a.v_pages, page * a.vp_page + (h0 + i) * a.vp_head + slot * a.vp_row + c);
    }
}

// Heads per lane: 4 share a token's angles and keep 128 bytes a lane in flight; 1 where that leaves fewer
// than two workgroups for each CU.
template <int DT, int D> int launch_append(const AppendArgs& a, const RotaryPlan& plan, hipStream_t s) {
    const int64_t blocks = ceil_div(a.tokens, 256 / (D / 8));
    const bool wide = blocks * ceil_div(a.heads, 4) >= 2 * device_compute_units();
    const int64_t groups = wide ? ceil_div(a.heads, 4) : a.heads;
    if (groups > 65535 || !fits_grid(blocks, 256)) return kUnsupportedShape;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
    if (wide) hipLaunchKernelGGL((append_pages_kernel<DT, D, 4>), grid, dim3(256), 0, s, a, plan);
    else hipLaunchKernelGGL((append_pages_kernel<DT, D, 1>), grid, dim3(256), 0, s, a, plan);
    return hipGetLastError();
}

}  // namespace
}  // namespace peco

using namespace peco;

PECO_API int peco_rotary_axes(const void* input, int64_t in_batch, int64_t in_head, int64_t in_row, void* output,
                              int64_t out_batch, int64_t out_head, int64_t out_row, const void* positions,
                              int position_type, int64_t position_batch, int64_t position_axis, const double* turns,
                              const int* axis_pairs, int axes, int halves, int inverse, int batch, int heads, int rows,
                              int dims, int dtype, void* stream) {
    RotaryPlan plan;
    if (!input || !output || batch < 1 || heads < 1 || rows < 1 ||
        !make_plan(plan, positions, position_type, position_batch, position_axis, turns, axis_pairs, axes, halves,
                   inverse, dims))
        return kInvalidValue;
    if (dims < 8 || dims > 512 || dims % 8) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return kUnsupportedDtype;
    const int64_t lanes = halves ? plan.pairs / 8 + (dims - 2 * plan.pairs) / 8 : dims / 8;
    if (static_cast<int64_t>(rows) * lanes > 0x7fffff00) return kUnsupportedShape;
    const int per16 = dtype == kF32 ? 4 : 8;  // elements in 16 bytes: every row of every head must start on them
    const int64_t strides = in_batch | in_head | in_row | out_batch | out_head | out_row;
    if (strides % per16 || reinterpret_cast<uintptr_t>(input) % 16 || reinterpret_cast<uintptr_t>(output) % 16)
        return kInvalidValue;
    RotaryArgs a{input,     output,   in_batch, in_head, in_row, out_batch, out_head,
                 out_row,   batch,    heads,    dims,    static_cast<uint32_t>(rows), static_cast<uint32_t>(lanes)};
    const auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case kBF16: return halves ? launch_rotary<kBF16, true>(a, plan, s) : launch_rotary<kBF16, false>(a, plan, s);
        case kF16: return halves ? launch_rotary<kF16, true>(a, plan, s) : launch_rotary<kF16, false>(a, plan, s);
        default: return halves ? launch_rotary<kF32, true>(a, plan, s) : launch_rotary<kF32, false>(a, plan, s);
    }
}

PECO_API int peco_append_pages(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* strides,
                               const int32_t* page_table, int64_t table_stride, const int32_t* offsets,
                               const int32_t* lengths, const void* positions, int position_type,
                               int64_t position_batch, int64_t position_axis, const double* turns,
                               const int* axis_pairs, int axes, int halves, int inverse, int batch, int heads,
                               int tokens, int pages, int page, int table_width, int dims, int dtype, void* stream) {
    RotaryPlan plan{};
    if (!k || !v || !k_pages || !v_pages || !strides || !page_table || !offsets || !lengths || batch < 1 || heads < 1 ||
        tokens < 1 || pages < 1 || page < 1 || table_width < 1 || table_stride < 0 ||
        (positions && !make_plan(plan, positions, position_type, 0, position_axis, turns, axis_pairs, axes, halves,
                                 inverse, dims)))
        return kInvalidValue;
    if (dims != 64 && dims != 128) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16) return kUnsupportedDtype;
    if (tokens > 0x3fffffff || static_cast<int64_t>(table_width) * page > 0x3fffffff) return kUnsupportedShape;
    int64_t all = 0;
    for (int i = 0; i < 10; ++i) all |= strides[i];
    for (const void* p : {k, v, static_cast<const void*>(k_pages), static_cast<const void*>(v_pages)})
        if (reinterpret_cast<uintptr_t>(p) % 16) return kInvalidValue;
    if (all % 8) return kInvalidValue;
    AppendArgs a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), static_cast<uint16_t*>(k_pages),
                 static_cast<uint16_t*>(v_pages), strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
                 strides[6], strides[7], strides[8], strides[9], page_table, offsets, lengths, table_stride, batch, heads,
                 tokens, pages, page, table_width, positions ? halves : 0};
    const auto s = static_cast<hipStream_t>(stream);
    if (dtype == kBF16) return dims == 128 ? launch_append<kBF16, 128>(a, plan, s) : launch_append<kBF16, 64>(a, plan, s);
    return dims == 128 ? launch_append<kF16, 128>(a, plan, s) : launch_append<kF16, 64>(a, plan, s);
}
