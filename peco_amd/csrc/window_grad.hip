// Attention with a sliding window and sinks: gradients.
//
// With P the weights, g the gradient of the output and delta_i = g_i . out_i (= sum_j P_ij dP_ij):
//   dV = P^T g,   dP = g V^T,   dS = P (dP - delta),   dQ = scale dS K,   dK = scale dS^T Q.
// P is computed again from Q, K and the forward's row statistics: P = 2^((s - m) scale log2 e - log2 l).
//
// Two launches (and the joins of walks that are cut), without atomics (every sum has one order):
//   dQ: a workgroup takes 128 rows as in the forward and walks their keys; per 32-key half S^T = K Q^T and
//       dP^T = V g^T (A = tile rows, B in registers), dQ^T += K^T dS^T (A = the K tile by transpose reads, B =
//       dS^T straight from the accumulators). It also forms delta, which the second launch reads.
//   dK/dV: a workgroup of 8 waves takes 256 keys, 32 a wave, and walks the rows that see any of them in 64-row
//       tiles of Q and g; S = Q K^T (B = K in registers) and dP = g V^T (B = V in LDS: with V in registers too the
//       sums of both leave room for one wave a SIMD only), dV^T += g^T P, dK^T += Q^T dS. The rows of all
//       query heads of the key head pass by, so shared heads need no further sum. Keys that are sinks are seen
//       by every later row: their walk is cut into parts, which a third launch adds up in order.
//
// S and dP are taken in both launches: seven products where five would do, but no atomics, and no gradient is read
// again. Measured with 128 channels, bf16, 24 heads of 7006 tokens in causal windows of 2026 with 256 sinks, calls in a
// row: dQ 261 us (946 TFLOP/s of its three products, MFMA busy 52% of the time), dK/dV 382 us (861 of its four, 45%), its
// join 7 us.
// Neither has LDS bank conflicts; what is left is the waves' waiting for LDS operands and for one another at the tiles'
// ends. 4 waves of 64 keys, which read half as much from LDS, took half as long again for dK/dV (one wave a SIMD covers
// nothing).
//
// Roundings: scores, dP, P and all sums are fp32; P and dS are rounded to the type for the products. delta takes out
// with what its rounding left: where a query sees a few keys dS is a small difference, and out's rounding alone
// would put as much error into it as dS's own.
// Fine calls (fine_call: few keys a query, or little work) go by kernels of their own: weights and dS enter their
// products as sums of two 16-bit numbers, and the weights' sum and delta are taken anew from fp32 weights by a first
// walk of dQ's, so that the results' own rounding is what is left.
// fp16: its smallest normal number, 2^-14, is large for a weight among thousands and for a gradient, so P enters
// its product times 2^14 and dS times a power of two taken from |dS| <= 2 max|g_i| max|V_j| (lengths of rows); both
// are divided out of the fp32 sums. bf16 has fp32's exponents and needs neither.
#include "window.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace peco {
namespace {

constexpr int kGradWaves = 8;               // of a dK/dV workgroup
constexpr int kGradKeys = 32 * kGradWaves;  // its keys
constexpr int kGradTile = 64;               // query rows of its tiles

struct GradArgs {
    const uint16_t *q, *k, *v, *out, *out_rest, *grad;
    uint16_t *dq, *dk, *dv;
    Strides qs, ks, vs, os, gs, dqs, dks, dvs;
    int heads, group, batch, queries, keys, left, right, sinks;
    float scale_log2, scale;
    const int32_t* lengths;
    const float *row_max, *row_log;  // [batch, query heads, queries]
    float* delta;                    // the same shape
    bool fine;
    float* fine_log;                 // fine: log2 of the sums of fp32 weights, the same shape
    int row_tiles, key_tiles, v_blocks;  // tiles of kWinRows rows, of kGradKeys keys, blocks of kWinRows keys
    int row_parts;                       // of every row tile's walk
    float* row_part;                     // dQ of each part [row_parts, query rows, D]
    // fp16: longest rows (squared) of V, per block of kWinRows of a key head, and of g, per row tile of one
    float *v_long, *g_long;
    int sink_tiles, sink_parts, parts;  // key tiles that hold sinks come first; parts of their walks and of the others'
    float* part;                        // [batch * heads, partial items, kGradKeys, 2, D]
};

// What the rounding of two packed values left.
template <int DT> __device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t packed) {
    return Mfma<DT>::pack2(a - half_to_f32<DT>(static_cast<uint16_t>(packed)),
                           b - half_to_f32<DT>(static_cast<uint16_t>(packed >> 16)));
}

enum Walk : int { kPlainWalk, kCarefulWalk, kSumsWalk };

struct Sequence {
    int queries, keys, position0;
};
__device__ __forceinline__ Sequence sequence_of(const GradArgs& A, int b) {
    Sequence s{A.queries, A.keys, A.keys - A.queries};
    if (A.lengths) {
        s.keys = s.queries = __builtin_amdgcn_readfirstlane(max(0, min(A.lengths[b], A.keys)));
        s.position0 = 0;
    }
    return s;
}

// A row's length for the bound on dS. A row with an infinity or NaN is left out: its dS is none that a factor could keep
// in range, and the other rows' keep theirs.
__device__ __forceinline__ float finite_length(float sq) { return sq < INFINITY ? sq : 0.0f; }

// fp16: dS is multiplied by this power of two (never more than 2^14 then).
__device__ __forceinline__ float dscale(float g2, float v2) {
    const float bound = 2.0f * sqrtf(g2) * sqrtf(v2);
    if (!(bound > 0x1p-80f && bound < 0x1p80f)) return 1.0f;
    int e;
    frexpf(bound, &e);  // bound < 2^e
    return ldexpf(1.0f, 14 - e);
}

template <int n> __device__ __forceinline__ float block_max(float v, float* tmp) {
#pragma unroll
    for (int m = kWave / 2; m; m /= 2) v = fmaxf(v, __shfl_xor(v, m, kWave));
    __syncthreads();
    if (threadIdx.x % kWave == 0) tmp[threadIdx.x / kWave] = v;
    __syncthreads();
    v = tmp[0];
#pragma unroll
    for (int i = 1; i < n; ++i) v = fmaxf(v, tmp[i]);
    return v;
}

// fp16: the longest of each block of kWinRows rows of V.
template <int D> __global__ __launch_bounds__(256) void value_lengths_kernel(GradArgs A) {
    __shared__ float tmp[4];
    const int bh = blockIdx.x / A.v_blocks, tile = blockIdx.x % A.v_blocks;
    const int b = bh / A.heads;
    const Sequence q = sequence_of(A, b);
    constexpr int G = D / 8;
    float most = 0.0f;
    for (int r = threadIdx.x / G; r < kWinRows; r += 256 / G) {
        const int key = tile * kWinRows + r;
        float sq = 0.0f;
        if (key < q.keys) {
            const u16x8 x = *reinterpret_cast<const u16x8*>(A.v + b * A.vs.b + (bh % A.heads) * A.vs.h +
                                                            static_cast<int64_t>(key) * A.vs.s + 8 * (threadIdx.x % G));
#pragma unroll
            for (int k = 0; k < 8; ++k) sq += f16_bits_to_f32(x[k]) * f16_bits_to_f32(x[k]);
        }
#pragma unroll
        for (int m = G / 2; m; m /= 2) sq += __shfl_xor(sq, m, kWave);
        most = fmaxf(most, finite_length(sq));
    }
    most = block_max<4>(most, tmp);
    if (threadIdx.x == 0) A.v_long[blockIdx.x] = most;
}

template <int DT, int D, bool kFar, bool kFine>
__global__ __launch_bounds__(256, 2) void window_dq_kernel(GradArgs A) {
    using T = WinTile<D>;
    constexpr int S = D / 16, NB = D / 32;
    __shared__ __align__(256) uint16_t kvs[4][T::kElems];  // K tiles, V tiles
    uint16_t(*const ks)[T::kElems] = kvs;
    uint16_t(*const vs)[T::kElems] = kvs + 2;
    __shared__ float tmp[4];

    // Parts of one row tile are as many workgroups apart as there are row tiles.
    const int heads = A.batch * A.heads, items = heads * A.row_tiles;
    const int part = static_cast<int>(blockIdx.x / items), item = static_cast<int>(blockIdx.x % items);
    const int bh = item % heads, tile = A.row_tiles - 1 - item / heads;
    const int b = bh / A.heads, kvh = bh % A.heads;
    const Sequence q = sequence_of(A, b);
    const int row0 = tile * kWinRows, rows = min(kWinRows, A.queries * A.group - row0);
    const int tid = threadIdx.x, lane = tid % kWave, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const bool wave_active = wave * 32 < rows;
    const bool qvalid = wave * 32 + lane % 32 < rows;
    const int lrow = min(row0 + wave * 32 + lane % 32, row0 + rows - 1);
    const int token = lrow / A.group, head = kvh * A.group + (lrow - token * A.group);
    const bool takes = qvalid && token < q.queries;

    const int t_first = row0 / A.group, t_last = min((row0 + rows - 1) / A.group, q.queries - 1);
    const KeyStream stream = t_first > t_last ? KeyStream{0, 0, 0}
                                              : key_stream(q.position0 + t_first, q.position0 + t_last, q.keys, A.left,
                                                           A.right, A.sinks);
    const int L = stream.length, l_last = max(L - 1, 0);
    const int all_tiles = static_cast<int>(ceil_div(L, kWinTile));
    const int per = static_cast<int>(ceil_div(all_tiles, A.row_parts));
    const int tile0 = min(part * per, all_tiles), tile1 = min(tile0 + per, all_tiles);
    const int pos = q.position0 + token;
    const int last_r = takes ? min(min(pos + A.right, q.keys - 1) - stream.delta, L - 1) : -1;
    const int first_r = pos - A.left - stream.delta;
    const int w_tok0 = min(row0 + wave * 32, row0 + rows - 1) / A.group;
    const int w_tok1 = min(row0 + wave * 32 + 31, row0 + rows - 1) / A.group;
    const int w_last =
        w_tok1 < q.queries ? min(min(q.position0 + w_tok0 + A.right, q.keys - 1) - stream.delta, L - 1) : -1;
    const int w_first = q.position0 + w_tok1 - A.left - stream.delta;
    const int w_any = min(min(q.position0 + w_tok1 + A.right, q.keys - 1) - stream.delta, L - 1);
    const int w_from = q.position0 + w_tok0 - A.left - stream.delta;

    // This lane's half of its query's rows: channels 16 s + 8 h .. + 7.
    u16x8 qf[S], gf[S];
    const int64_t row_id = (static_cast<int64_t>(b) * (A.heads * A.group) + head) * A.queries + token;
    float delta = 0.0f, g2 = 0.0f;
    {
        const uint16_t* qrow = A.q + b * A.qs.b + head * A.qs.h + token * A.qs.s;
        const uint16_t* grow = A.grad + b * A.gs.b + head * A.gs.h + token * A.gs.s;
        const uint16_t* orow = A.out + b * A.os.b + head * A.os.h + token * A.os.s;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            qf[s] = *reinterpret_cast<const u16x8*>(qrow + 16 * s + 8 * h);
            gf[s] = *reinterpret_cast<const u16x8*>(grow + 16 * s + 8 * h);
            const u16x8 of = *reinterpret_cast<const u16x8*>(orow + 16 * s + 8 * h);
            const u16x8 rest = *reinterpret_cast<const u16x8*>(A.out_rest + row_id * D + 16 * s + 8 * h);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float g = half_to_f32<DT>(gf[s][k]);
                delta += g * (half_to_f32<DT>(of[k]) + half_to_f32<DT>(rest[k]));
                if constexpr (DT == kF16) g2 += g * g;
            }
        }
    }
    delta += __shfl_xor(delta, 32, kWave);
    if (!takes) delta = 0.0f;
    if (!kFine && qvalid && h == 0 && part == 0) A.delta[row_id] = delta;
    float dmul = 1.0f;
    if constexpr (DT == kF16) {
        g2 += __shfl_xor(g2, 32, kWave);
        if (!takes) g2 = 0.0f;
        g2 = finite_length(g2);
        const float longest = block_max<4>(g2, tmp);
        if (tid == 0 && part == 0) A.g_long[static_cast<int64_t>(bh) * A.row_tiles + tile] = longest;
        float v2 = 0.0f;
        for (int i = tid; i < A.v_blocks; i += 256) v2 = fmaxf(v2, A.v_long[static_cast<int64_t>(bh) * A.v_blocks + i]);
        dmul = dscale(g2, block_max<4>(v2, tmp));
    }
    // (A row that sees nothing has the lowest float and an infinite sum: weights of 0.) fp16: dS's factor is a power of
    // two and goes into its weight's exponent.
    const float m = A.row_max[row_id];
    float log_l = A.row_log[row_id];
    if constexpr (!kFine && DT == kF16) log_l -= log2f(dmul);
    const bool own_wide = m != -FLT_MAX && fabsf(m * A.scale_log2) > kWideScores, wide = __any(own_wide);
    float offset = own_wide ? -log_l : __builtin_fmaf(-m, A.scale_log2, -log_l);

    const uint16_t* kh = A.k + b * A.ks.b + kvh * A.ks.h;
    const uint16_t* vh = A.v + b * A.vs.b + kvh * A.vs.h;
    auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
            const int span = i * 4 + wave;
            const int r = span * T::kWaveRows + lane / T::CH, p = lane % T::CH;
            const uint32_t chunk = (p ^ T::swz(r)) * 16;
            const int sr = min(t * kWinTile + r, l_last);
            load_row16<kFar>(kh, sr < stream.a1 ? sr : sr + stream.delta, A.ks.s, chunk, lds_addr(ks[buf] + span * kWave * 8));
            load_row16<kFar>(vh, sr < stream.a1 ? sr : sr + stream.delta, A.vs.s, chunk, lds_addr(vs[buf] + span * kWave * 8));
        }
#endif
    };
    f32x16 acc[NB];
    [[maybe_unused]] float sum_p = 0.0f, sum_pdp = 0.0f;
    const WinLane<D> at(lane, kvs[0]);
    auto compute = [&](auto kind, int t, int buf, int cb) __attribute__((always_inline)) {
        const int kt = 2 * (buf * T::kElems + 32 * cb * D), vt = kt + 4 * T::kElems;  // bytes from the first tile
        const int r0 = t * kWinTile + 32 * cb;
        if (r0 > w_any || (r0 + 31 < w_from && r0 >= A.sinks)) {
            return;
        }
        const bool whole = r0 + 31 <= w_last && (r0 >= w_first || r0 + 31 < A.sinks);
        f32x16 sacc{}, pacc{};
#pragma unroll
        for (int s = 0; s < S; ++s) {  // in turn: two chains, each product behind the other chain's
            sacc = Mfma<DT>::run(at.rows(kt, s), qf[s], sacc);
            pacc = Mfma<DT>::run(at.rows(vt, s), gf[s], pacc);
        }
        read_ahead<2 * S, 2 * S, 4>();
        __builtin_amdgcn_sched_barrier(0);
        auto seen_at = [&](int row) {
            const int r = r0 + row;
            return r <= last_r && (r >= first_r || r < A.sinks);
        };
        if (wide) {  // (for the queries that need it: the others' weights keep their bits)
            const float reference = own_wide ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sacc[i] -= reference;
        }
        if constexpr (decltype(kind)::value == kSumsWalk) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i], A.scale_log2, offset));
                const bool seen = whole || seen_at(8 * (i / 4) + 4 * h + i % 4);
                sum_p += seen ? p : 0.0f;
                sum_pdp += seen ? p * pacc[i] : 0.0f;
            }
            return;
        }
        float ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i], A.scale_log2, offset));
            ds[i] = p * (pacc[i] - delta);
        }
        if (!whole) {
            // (Element i is row 8 (i / 4) + 4 h + i % 4: the lane's 4 h is taken off the limits, the rest is uniform.)
            const int last = last_r - 4 * h, from = first_r - 4 * h, sinks = A.sinks - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = r0 + 8 * (i / 4) + i % 4;
                if (!(r <= last && (r >= from || r < sinks))) ds[i] = 0.0f;
            }
        }
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = Mfma<DT>::pack2(ds[2 * i], ds[2 * i + 1]);
        auto add = [&]() __attribute__((always_inline)) {
            if constexpr (decltype(kind)::value == kCarefulWalk) {
                if (!whole && rows_not_finite<DT, D>(kvs[0], kt, lane)) {
                    add_rows_seen<DT, D>(acc, kt, w, at, h, seen_at);
                    return;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            add_rows<DT, D>(acc, kt, w, at);
        };
        add();
        if constexpr (kFine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = rest2<DT>(ds[2 * i], ds[2 * i + 1], w[i]);
            add();
        }
    };
    auto walk = [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x16{};
        if (tile0 >= tile1) return;
#if defined(__HIP_DEVICE_COMPILE__)
        // (What the loop reads from registers has arrived: the compiler does not count the tile loads.)
#pragma unroll
        for (int s = 0; s < S; ++s) asm volatile("" ::"v"(qf[s]), "v"(gf[s]));
        asm volatile("" ::"v"(m), "v"(offset));
#endif
        load_tile(tile0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        auto step = [&](auto bufc, int t) __attribute__((always_inline)) {
            const int buf = bufc;
            if (t + 1 < tile1) load_tile(t + 1, buf ^ 1);
            if (!wave_active) {
            } else if constexpr (decltype(kind)::value != kPlainWalk) {
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) compute(kind, t, buf, cb);
            } else {
                compute(kind, t, buf, 0);
                compute(kind, t, buf, 1);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        };
        if constexpr (decltype(kind)::value != kPlainWalk) {
#pragma unroll 1
            for (int t = tile0; t < tile1; ++t) step((t - tile0) & 1, t);
        } else {
            for (int t = tile0; t < tile1; t += 2) {
                step(std::integral_constant<int, 0>{}, t);
                if (t + 1 < tile1) step(std::integral_constant<int, 1>{}, t + 1);
            }
        }
    };
    if constexpr (kFine) {
        // (A walk that is cut is long: its weights' roundings have averaged out in the forward's sum and output.)
        if (A.row_parts == 1) {
            walk(std::integral_constant<int, kSumsWalk>{});
            sum_p += __shfl_xor(sum_p, 32, kWave);
            sum_pdp += __shfl_xor(sum_pdp, 32, kWave);
            if (sum_p != 0.0f) {  // (a row that sees nothing keeps its infinite sum)
                delta = sum_pdp / sum_p;
                log_l += log2f(sum_p);
            }
        }
        if (qvalid && h == 0 && part == 0) {
            A.delta[row_id] = delta;
            A.fine_log[row_id] = log_l;
        }
        if constexpr (DT == kF16) log_l -= log2f(dmul);
        offset = own_wide ? -log_l : __builtin_fmaf(-m, A.scale_log2, -log_l);
    }
    walk(std::integral_constant<int, kPlainWalk>{});
    if (__syncthreads_or(wave_active && !all_finite(acc))) walk(std::integral_constant<int, kCarefulWalk>{});
    if (!qvalid) return;
    const float mul = A.scale / dmul;
    if (A.row_parts > 1) {
        const int64_t rows_all = static_cast<int64_t>(heads) * A.group * A.queries;
        float* o = A.row_part + (part * rows_all + row_id) * D;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x{acc[nb][4 * g] * mul, acc[nb][4 * g + 1] * mul, acc[nb][4 * g + 2] * mul, acc[nb][4 * g + 3] * mul};
                *reinterpret_cast<f32x4*>(o + 32 * nb + 8 * g + 4 * h) = takes ? x : f32x4{};
            }
        return;
    }
    uint16_t* o = A.dq + b * A.dqs.b + head * A.dqs.h + token * A.dqs.s;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t w0 = Mfma<DT>::pack2(acc[nb][4 * g] * mul, acc[nb][4 * g + 1] * mul);
            const uint32_t w1 = Mfma<DT>::pack2(acc[nb][4 * g + 2] * mul, acc[nb][4 * g + 3] * mul);
            *reinterpret_cast<u32x2*>(o + 32 * nb + 8 * g + 4 * h) = takes ? u32x2{w0, w1} : u32x2{0, 0};
        }
}

// dQ of the row tiles whose walks were cut: the parts' sums, in order. D / 4 lanes a row.
template <int DT, int D> __global__ __launch_bounds__(256) void window_dq_join_kernel(GradArgs A) {
    constexpr int kLanes = D / 4;
    const int hq = A.heads * A.group;
    const int64_t rows_all = static_cast<int64_t>(A.batch) * hq * A.queries;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
    if (row >= rows_all) return;
    const int c = 4 * (threadIdx.x % kLanes);
    f32x4 sum{};
    for (int i = 0; i < A.row_parts; ++i) sum += *reinterpret_cast<const f32x4*>(A.row_part + (i * rows_all + row) * D + c);
    const int64_t token = row % A.queries, head = row / A.queries % hq, b = row / A.queries / hq;
    *reinterpret_cast<u32x2*>(A.dq + b * A.dqs.b + head * A.dqs.h + token * A.dqs.s + c) =
        u32x2{Mfma<DT>::pack2(sum[0], sum[1]), Mfma<DT>::pack2(sum[2], sum[3])};
}

// Items of a head: the sink tiles' parts, then the other tiles' parts.
__host__ __device__ __forceinline__ int64_t grad_items(const GradArgs& A) {
    return static_cast<int64_t>(A.sink_tiles) * A.sink_parts + static_cast<int64_t>(A.key_tiles - A.sink_tiles) * A.parts;
}
// Items of a head whose results are partial (the first ones of the list).
__host__ __device__ __forceinline__ int64_t partial_items(const GradArgs& A) {
    if (A.parts > 1) return grad_items(A);
    return A.sink_parts > 1 ? static_cast<int64_t>(A.sink_tiles) * A.sink_parts : 0;
}

template <int DT, int D, bool kFine>
__global__ __launch_bounds__(kGradWaves * kWave, 2) void window_dkv_kernel(GradArgs A) {
    using T = WinTile<D>;
    constexpr int S = D / 16, NB = D / 32;
    constexpr int kTile = kGradTile, kElems = kTile * D, kLoads = kTile / (kGradWaves * T::kWaveRows);
    __shared__ __align__(256) uint16_t tiles_lds[4][kElems];  // Q tiles, g tiles
    uint16_t(*const qt_)[kElems] = tiles_lds;
    uint16_t(*const gt_)[kElems] = tiles_lds + 2;
    // Operands of the workgroup's keys, as each lane takes them: V, and the last kSpilled steps of K. (With all of K
    // in registers the compiler spills some of it to memory, whose loads wait for the tile loads before them.)
    constexpr int kSpilled = D == 128 ? 3 : 0, kHeld = S - kSpilled;
    __shared__ u16x8 operands[kGradWaves][S + kSpilled][kWave];
    __shared__ __align__(16) float stat[2][3][kTile];  // references, log2 sums and deltas of a tile's rows
    __shared__ float tmp[kGradWaves];

    const int heads = A.batch * A.heads;
    const int bh = blockIdx.x % heads;
    const int item = static_cast<int>(blockIdx.x / heads);
    const int sink_items = A.sink_tiles * A.sink_parts;
    const bool sink = item < sink_items;
    const int parts = sink ? A.sink_parts : A.parts;
    const int tile = sink ? item / parts : A.sink_tiles + (item - sink_items) / parts;
    const int part = sink ? item % parts : (item - sink_items) % parts;
    const int b = bh / A.heads, kvh = bh % A.heads;
    const Sequence q = sequence_of(A, b);
    const int tid = threadIdx.x, lane = tid % kWave, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int key0 = tile * kGradKeys, wkey0 = key0 + 32 * wave;
    const int key = wkey0 + lane % 32;  // this lane's column

    // Rows of the stream that see key j: [row_from(j), row_to(j)).
    const int all_rows = q.queries * A.group;
    auto row_from = [&](int j) {
        const int64_t t = max(static_cast<int64_t>(j) - A.right - q.position0, int64_t{0});
        return static_cast<int>(min(t * A.group, static_cast<int64_t>(all_rows)));
    };
    auto row_to = [&](int j) {
        const int64_t t = j < A.sinks ? int64_t{1} << 31 : static_cast<int64_t>(j) + A.left - q.position0 + 1;
        return static_cast<int>(max(min(t * A.group, static_cast<int64_t>(all_rows)), int64_t{0}));
    };
    const int last_key = min(key0 + kGradKeys, q.keys) - 1;
    int r_begin = 0, r_end = 0;
    if (last_key >= key0) {
        r_begin = row_from(key0);
        r_end = key0 < A.sinks ? all_rows : row_to(last_key);
    }
    // Tiles of this part.
    const int all_tiles = r_end > r_begin ? static_cast<int>(ceil_div(r_end - r_begin, kTile)) : 0;
    const int per = static_cast<int>(ceil_div(all_tiles, parts));
    const int tile0 = min(part * per, all_tiles), tile1 = min(tile0 + per, all_tiles);
    const bool held = key < q.keys;
    const int from = held ? row_from(key) : 0x7fffffff, to = held ? row_to(key) : 0;
    // Of the wave's keys: every one is seen by the rows [w_from, w_to), none by rows outside [w_first, w_last).
    const bool wave_active = wkey0 < q.keys;
    const int wlast = min(wkey0 + 31, q.keys - 1);
    const int w_from = wkey0 + 31 < q.keys ? row_from(wlast) : 0x7fffffff, w_to = row_to(wkey0 + 31 < A.sinks ? wkey0 : max(wkey0, A.sinks));
    const int w_first = row_from(wkey0), w_last = wkey0 < A.sinks ? all_rows : row_to(wlast);

    u16x8 kf[kHeld];
    {
        const int row = min(key, A.keys - 1);
        const uint16_t* krow = A.k + b * A.ks.b + kvh * A.ks.h + row * A.ks.s;
        const uint16_t* vrow = A.v + b * A.vs.b + kvh * A.vs.h + row * A.vs.s;
        u16x8(*const own)[kWave] = operands[wave];  // (a wave reads what it wrote: no barrier)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            own[s][lane] = *reinterpret_cast<const u16x8*>(vrow + 16 * s + 8 * h);
            const u16x8 x = *reinterpret_cast<const u16x8*>(krow + 16 * s + 8 * h);
            if (s < kHeld) kf[s] = x;
            else own[S + s - kHeld][lane] = x;
        }
    }
    float dmul = 1.0f;
    if constexpr (DT == kF16) {
        float g2 = 0.0f, v2 = 0.0f;
        for (int i = tid; i < A.row_tiles; i += kGradWaves * kWave) g2 = fmaxf(g2, A.g_long[static_cast<int64_t>(bh) * A.row_tiles + i]);
        for (int i = tid; i < A.v_blocks; i += kGradWaves * kWave) v2 = fmaxf(v2, A.v_long[static_cast<int64_t>(bh) * A.v_blocks + i]);
        g2 = block_max<kGradWaves>(g2, tmp);
        dmul = dscale(g2, block_max<kGradWaves>(v2, tmp));
    }

    const uint16_t* qh = A.q + b * A.qs.b + static_cast<int64_t>(kvh) * A.group * A.qs.h;
    const uint16_t* gh = A.grad + b * A.gs.b + static_cast<int64_t>(kvh) * A.group * A.gs.h;
    const int64_t stat0 = (static_cast<int64_t>(b) * A.heads + kvh) * A.group * A.queries;
    auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int first = r_begin + t * kTile;
        int lane = threadIdx.x % kWave;
        asm volatile("" : "+v"(lane));  // (the lane's shares of the addresses are computed again, not held)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int span = i * kGradWaves + wave;
            const int r = span * T::kWaveRows + lane / T::CH, p = lane % T::CH;
            const int chunk = (p ^ T::swz(r)) * 8;
            const int row = min(first + r, r_end - 1);  // rows past the walk repeat its last row
            const int token = A.group == 1 ? row : row / A.group, head = row - token * A.group;
            dma16(qh + head * A.qs.h + token * A.qs.s + chunk, lds_addr(qt_[buf] + span * kWave * 8));
            dma16(gh + head * A.gs.h + token * A.gs.s + chunk, lds_addr(gt_[buf] + span * kWave * 8));
        }
        if (wave < 3 && lane < kTile) {
            const int row = min(first + lane, r_end - 1);
            const int token = A.group == 1 ? row : row / A.group, head = row - token * A.group;
            const float* from = wave == 0 ? A.row_max : wave == 2 ? A.delta : kFine ? A.fine_log : A.row_log;
            dma4(from + stat0 + static_cast<int64_t>(head) * A.queries + token, lds_addr(stat[buf][wave]));
        }
#endif
    };

    f32x16 dk[NB], dv[NB];
    const WinLane<D> at0(lane, tiles_lds[0]);
    // One 32-row half of a tile: S and P, then dV, then dP and dS, then dK, which keeps one 32 x 32 result and its packed form alive
    // at a time beside the sums.
    auto compute = [&](auto careful, int t, int buf, int cb) __attribute__((always_inline)) {
        const int qoff = 2 * (buf * kElems + 32 * cb * D), goff = qoff + 4 * kElems;  // bytes from the first tile
        constexpr int qt = 0, gt = 4 * kElems;  // (`at` holds the buffer and the half)
        const int r0 = r_begin + t * kTile + 32 * cb;
        if (r0 + 31 < w_first || r0 >= w_last) return;
        const bool whole = r0 >= w_from && r0 + 31 < w_to;
        [[maybe_unused]] const bool one_by_one =
            decltype(careful)::value && !whole &&
            (rows_not_finite<DT, D>(tiles_lds[0], qoff, lane) || rows_not_finite<DT, D>(tiles_lds[0], goff, lane));
        auto seen_at = [&](int row) { return r0 + row >= from && r0 + row < to; };
        f32x16 p{}, ds{};
        WinLane<D> at = at0.moved(qoff);
        at.fresh();
        // (The channels in the forward's order: the references and sums are those of its scores, and where scores are
        // large another order's rounding moves the exponents.)
#pragma unroll
        for (int s = 0; s < S; ++s)
            p = Mfma<DT>::run(at.rows(qt, s), s < kHeld ? kf[s < kHeld ? s : 0] : operands[wave][S + s - kHeld][lane], p);
        read_ahead<S, S + kSpilled, 6>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 m = *reinterpret_cast<const f32x4*>(&stat[buf][0][32 * cb + 8 * g + 4 * h]);
            const f32x4 log_l = *reinterpret_cast<const f32x4*>(&stat[buf][1][32 * cb + 8 * g + 4 * h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __builtin_fmaf(p[4 * g + i] - m[i], A.scale_log2, DT == kF16 ? 14.0f - log_l[i] : -log_l[i]);
                p[4 * g + i] = __builtin_amdgcn_exp2f(x);  // (fp16: times 2^14)
            }
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = r0 + 8 * (i / 4) + i % 4;
                if (!(r >= from - 4 * h && r < to - 4 * h)) p[i] = 0.0f;
            }
        }
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = Mfma<DT>::pack2(p[2 * i], p[2 * i + 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (one_by_one) add_rows_seen<DT, D>(dv, gt, w, at, h, seen_at);
        else add_rows<DT, D>(dv, gt, w, at);
        if constexpr (kFine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = rest2<DT>(p[2 * i], p[2 * i + 1], w[i]);
            if (one_by_one) add_rows_seen<DT, D>(dv, gt, w, at, h, seen_at);
            else add_rows<DT, D>(dv, gt, w, at);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < S; ++s) ds = Mfma<DT>::run(at.rows(gt, s), operands[wave][s][lane], ds);
        read_ahead<S, 2 * S, 6>();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 delta = *reinterpret_cast<const f32x4*>(&stat[buf][2][32 * cb + 8 * g + 4 * h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ds[4 * g + i] = p[4 * g + i] * (ds[4 * g + i] - delta[i]);
                if constexpr (DT == kF16) ds[4 * g + i] *= dmul * 0x1p-14f;
            }
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = r0 + 8 * (i / 4) + i % 4;
                if (!(r >= from - 4 * h && r < to - 4 * h)) ds[i] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = Mfma<DT>::pack2(ds[2 * i], ds[2 * i + 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (one_by_one) add_rows_seen<DT, D>(dk, qt, w, at, h, seen_at);
        else add_rows<DT, D>(dk, qt, w, at);
        if constexpr (kFine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = rest2<DT>(ds[2 * i], ds[2 * i + 1], w[i]);
            if (one_by_one) add_rows_seen<DT, D>(dk, qt, w, at, h, seen_at);
            else add_rows<DT, D>(dk, qt, w, at);
        }
    };
    auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) dk[nb] = dv[nb] = f32x16{};
        if (tile0 >= tile1) return;
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int s = 0; s < kHeld; ++s) asm volatile("" ::"v"(kf[s]));
#endif
        load_tile(tile0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        auto step = [&](int buf, int t) __attribute__((always_inline)) {
            if (t + 1 < tile1) load_tile(t + 1, buf ^ 1);
            if (wave_active) {
#pragma unroll 1
                for (int cb = 0; cb < kTile / 32; ++cb) compute(careful, t, buf, cb);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        };
#pragma unroll 1
        for (int t = tile0; t < tile1; ++t) step((t - tile0) & 1, t);
    };
    walk(std::false_type{});
    if (__syncthreads_or(wave_active && !(all_finite(dk) && all_finite(dv)))) walk(std::true_type{});
    const float kmul = A.scale / dmul, vmul = DT == kF16 ? 0x1p-14f : 1.0f;
    if (parts > 1) {
        // [head, item, key, dK | dV, D]; every key of the tile, so that the join reads nothing unwritten.
        float* o = A.part + ((static_cast<int64_t>(bh) * partial_items(A) + item) * kGradKeys + 32 * wave + lane % 32) * 2 * D;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * nb + 8 * g + 4 * h;
                *reinterpret_cast<f32x4*>(o + d) = f32x4{dk[nb][4 * g] * kmul, dk[nb][4 * g + 1] * kmul,
                                                         dk[nb][4 * g + 2] * kmul, dk[nb][4 * g + 3] * kmul};
                *reinterpret_cast<f32x4*>(o + D + d) = f32x4{dv[nb][4 * g] * vmul, dv[nb][4 * g + 1] * vmul,
                                                             dv[nb][4 * g + 2] * vmul, dv[nb][4 * g + 3] * vmul};
            }
        return;
    }
    if (key >= A.keys) return;
    uint16_t* ok = A.dk + b * A.dks.b + kvh * A.dks.h + key * A.dks.s;
    uint16_t* ov = A.dv + b * A.dvs.b + kvh * A.dvs.h + key * A.dvs.s;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * nb + 8 * g + 4 * h;
            *reinterpret_cast<u32x2*>(ok + d) = u32x2{Mfma<DT>::pack2(dk[nb][4 * g] * kmul, dk[nb][4 * g + 1] * kmul),
                                                      Mfma<DT>::pack2(dk[nb][4 * g + 2] * kmul, dk[nb][4 * g + 3] * kmul)};
            *reinterpret_cast<u32x2*>(ov + d) = u32x2{Mfma<DT>::pack2(dv[nb][4 * g] * vmul, dv[nb][4 * g + 1] * vmul),
                                                      Mfma<DT>::pack2(dv[nb][4 * g + 2] * vmul, dv[nb][4 * g + 3] * vmul)};
        }
}

// dK and dV of the key tiles whose walks were cut: the parts' sums, in order. D / 2 lanes a key (4 values each of
// dK, then of dV).
template <int DT, int D> __global__ __launch_bounds__(256) void window_dkv_join_kernel(GradArgs A) {
    constexpr int kLanes = D / 2;
    const int heads = A.batch * A.heads;
    const int split_tiles = A.parts > 1 ? A.key_tiles : A.sink_tiles;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
    const int64_t per_head = static_cast<int64_t>(split_tiles) * kGradKeys;
    if (row >= heads * per_head) return;
    const int bh = static_cast<int>(row / per_head), key = static_cast<int>(row % per_head);
    const int tile = key / kGradKeys;
    if (key >= A.keys || (tile < A.sink_tiles ? A.sink_parts : A.parts) == 1) return;
    const bool sink = tile < A.sink_tiles;
    const int parts = sink ? A.sink_parts : A.parts;
    const int64_t item = sink ? static_cast<int64_t>(tile) * parts
                              : static_cast<int64_t>(A.sink_tiles) * A.sink_parts + static_cast<int64_t>(tile - A.sink_tiles) * parts;
    const int c = 4 * (threadIdx.x % kLanes);
    const float* p = A.part + ((static_cast<int64_t>(bh) * partial_items(A) + item) * kGradKeys + key % kGradKeys) * 2 * D + c;
    f32x4 sum{};
    for (int i = 0; i < parts; ++i) sum += *reinterpret_cast<const f32x4*>(p + static_cast<int64_t>(i) * kGradKeys * 2 * D);
    const int b = bh / A.heads, kvh = bh % A.heads;
    uint16_t* o = c < D ? A.dk + b * A.dks.b + kvh * A.dks.h + key * A.dks.s + c
                        : A.dv + b * A.dvs.b + kvh * A.dvs.h + key * A.dvs.s + (c - D);
    *reinterpret_cast<u32x2*>(o) = u32x2{Mfma<DT>::pack2(sum[0], sum[1]), Mfma<DT>::pack2(sum[2], sum[3])};
}

// Parts of the key tiles' walks. Under a window a tile without sinks is seen by about left + right + 256 tokens,
// one with sinks by every later token: the latter's walk is cut to about the former's length, so that no
// workgroup walks on alone, but to no less than a quarter of a CU's share of the call (where the sinks are many there
// are workgroups enough, and each part costs workspace).
// Calls of few key tiles cut the other walks too: a workgroup to a CU at a time, the rounds of workgroups times a
// part's tiles and a fixed cost, plus the third launch, which reads the parts' fp32 sums. Measured (128 channels: 3.3 us
// a tile and 15 fixed, 64 channels: 2.0 and 10): one head of 7006 tokens without a window (28 key tiles) 333 us uncut,
// 80 in 6 parts, 69 in 12; 24 heads of 1800 tokens in windows of 512 (192) 55 uncut, 86 in 2 parts; 8 heads of 777
// tokens in windows of 256 (32, 64 channels) 41 in 2 parts, 30 in 8.
constexpr int kGradPartTiles = 2;  // of a part at least
constexpr int kMaxParts = 64;

// Whether a call is a fine one. Roundings of weights, delta and dS leave the gradients 1.4 to 1.5 times as far off as
// their own rounding does; where a query sees few keys (weights are large, dS is a small difference) or rows are few
// (nothing averages out) it was up to 2, in a quarter of short sequences above 1.5. Fine calls are at 1.00. Measured,
// a captured step of forward and gradients, fine against not: 24 heads x 200 tokens 72 and 58 us (195 either way where
// the host makes the call), 1 x 1000 72 and 67, 24 x 7006 in windows of 32 keys 308 and 256: larger calls only where
// they need it, with up to 8 keys (at 16 and more the others are below 1.5).
constexpr int kFineKeys = 8;
constexpr int64_t kFinePairs = 1 << 20;
bool fine_call(const GradArgs& A) {
    const int64_t most = std::min<int64_t>(A.keys, int64_t{A.left} + A.right + 1 + A.sinks);  // keys that a query may see
    return most <= kFineKeys || int64_t{A.batch} * A.heads * A.group * A.queries <= kFinePairs / most;
}

void plan_parts(GradArgs& A, int d) {
    A.fine = fine_call(A);
    A.row_tiles = static_cast<int>(ceil_div(static_cast<int64_t>(A.queries) * A.group, kWinRows));
    A.key_tiles = static_cast<int>(ceil_div(A.keys, kGradKeys));
    A.v_blocks = static_cast<int>(ceil_div(A.keys, kWinRows));
    const int64_t tokens = std::min<int64_t>(A.queries, kWinRows / A.group + 1);
    A.row_parts = cut_parts(static_cast<int64_t>(A.batch) * A.heads * A.row_tiles,
                            seen_keys(A.keys, tokens, A.left, A.right, A.sinks),
                            static_cast<int64_t>(A.batch) * A.heads * A.group * A.queries, d);
    const int64_t all = ceil_div(static_cast<int64_t>(A.queries) * A.group, kGradTile);
    const int64_t window = std::min<int64_t>(A.queries, static_cast<int64_t>(A.left) + A.right + kGradKeys);
    const int64_t walk = std::max<int64_t>(1, std::min(all, ceil_div(window * A.group, kGradTile)));
    A.sink_tiles = static_cast<int>(std::min<int64_t>(A.key_tiles, ceil_div(A.sinks, kGradKeys)));
    const int64_t items = static_cast<int64_t>(A.batch) * A.heads * A.key_tiles;
    const int64_t slots = device_compute_units();
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMaxParts, walk / kGradPartTiles));
    const double tile_us = d == 128 ? 3.3 : 2.0, fixed_us = d == 128 ? 15.0 : 10.0;
    double least = 1e30;
    A.parts = 1;
    for (int n = 1; n <= most; ++n) {
        double cost = static_cast<double>(ceil_div(items * n, slots)) * (fixed_us + tile_us * static_cast<double>(ceil_div(walk, n)));
        if (n > 1) cost += 4.0 + static_cast<double>(items) * n * kGradKeys * 2 * d * 4 / 6.0e6;  // 4 us and 6 TB/s
        if (cost >= least) continue;
        least = cost;
        A.parts = n;
    }
    const int64_t total = static_cast<int64_t>(A.batch) * A.heads *
                          (A.sink_tiles * all + (A.key_tiles - A.sink_tiles) * walk);
    const int64_t per =
        std::max({int64_t{kGradPartTiles}, ceil_div(walk, A.parts), ceil_div(total, 4 * slots)});
    A.sink_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxParts, ceil_div(all, per))));
    if (A.sink_tiles == 0) A.sink_parts = 1;
}

struct GradLayout {
    int64_t fine_log, v_long, g_long, part, floats;  // (delta is at 0)
};
GradLayout grad_layout(const GradArgs& A, int d, int dtype) {
    const int64_t heads = static_cast<int64_t>(A.batch) * A.heads;
    auto up = [](int64_t n) { return ceil_div(n, 4) * 4; };
    GradLayout l{};
    l.fine_log = up(heads * A.group * A.queries);
    l.v_long = l.fine_log * (A.fine ? 2 : 1);
    l.g_long = l.v_long + (dtype == kF16 ? up(heads * A.v_blocks) : 0);
    l.part = l.g_long + (dtype == kF16 ? up(heads * A.row_tiles) : 0);
    // (One after the other: the parts of dQ are joined before the next launch writes its own.)
    const int64_t row_parts = A.row_parts > 1 ? A.row_parts * heads * A.group * A.queries * d : 0;
    l.floats = l.part + std::max(row_parts, heads * partial_items(A) * kGradKeys * 2 * d);
    return l;
}

template <int DT, int D, bool kFine> int launch_grad(const GradArgs& A, bool far, hipStream_t s) {
    const int64_t heads = static_cast<int64_t>(A.batch) * A.heads;
    const int64_t dq = heads * A.row_tiles * A.row_parts, dkv = heads * grad_items(A);
    const int64_t dq_join = A.row_parts > 1 ? ceil_div(heads * A.group * A.queries, 256 / (D / 4)) : 0;
    const int64_t joined = heads * (A.parts > 1 ? A.key_tiles : A.sink_tiles) * kGradKeys;
    const int64_t dkv_join = partial_items(A) ? ceil_div(joined, 256 / (D / 2)) : 0;
    // (Before the first launch: a call runs whole or not at all.)
    if (!fits_grid(std::max({dq, heads * A.v_blocks, dq_join, dkv_join}), 256) || !fits_grid(dkv, kGradWaves * kWave))
        return kUnsupportedShape;
    if constexpr (DT == kF16)
        hipLaunchKernelGGL((value_lengths_kernel<D>), dim3(static_cast<unsigned>(heads * A.v_blocks)), dim3(256), 0, s, A);
    if (far) hipLaunchKernelGGL((window_dq_kernel<DT, D, true, kFine>), dim3(static_cast<unsigned>(dq)), dim3(256), 0, s, A);
    else hipLaunchKernelGGL((window_dq_kernel<DT, D, false, kFine>), dim3(static_cast<unsigned>(dq)), dim3(256), 0, s, A);
    if (dq_join)
        hipLaunchKernelGGL((window_dq_join_kernel<DT, D>), dim3(static_cast<unsigned>(dq_join)), dim3(256), 0, s, A);
    hipLaunchKernelGGL((window_dkv_kernel<DT, D, kFine>), dim3(static_cast<unsigned>(dkv)), dim3(kGradWaves * kWave), 0, s, A);
    if (dkv_join)
        hipLaunchKernelGGL((window_dkv_join_kernel<DT, D>), dim3(static_cast<unsigned>(dkv_join)), dim3(256), 0, s, A);
    return hipGetLastError();
}

template <int DT, int D> int launch_type(const GradArgs& A, bool far, hipStream_t s) {
    return A.fine ? launch_grad<DT, D, true>(A, far, s) : launch_grad<DT, D, false>(A, far, s);
}

Strides strides_of(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }
bool shape_ok(int batch, int q_heads, int kv_heads, int queries, int keys, int left, int right, int sinks) {
    return batch >= 1 && kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0 && queries >= 1 && keys >= 1 &&
           left >= -1 && right >= -1 && sinks >= 0 && left <= kUnbounded && right <= kUnbounded && sinks <= kUnbounded;
}
GradArgs sizes_of(int batch, int q_heads, int kv_heads, int queries, int keys, int left, int right, int sinks, int d) {
    GradArgs A{};
    A.batch = batch;
    A.heads = kv_heads;
    A.group = q_heads / kv_heads;
    A.queries = queries;
    A.keys = keys;
    A.left = left < 0 ? kUnbounded : left;
    A.right = right < 0 ? kUnbounded : right;
    A.sinks = sinks;
    plan_parts(A, d);
    return A;
}

}  // namespace
}  // namespace peco

using namespace peco;

PECO_API size_t peco_window_attention_grad_workspace_size(int batch, int q_heads, int kv_heads, int queries, int keys,
                                                          int left, int right, int sinks, int d, int dtype) {
    if (!shape_ok(batch, q_heads, kv_heads, queries, keys, left, right, sinks)) return 0;
    return static_cast<size_t>(
        grad_layout(sizes_of(batch, q_heads, kv_heads, queries, keys, left, right, sinks, d), d, dtype).floats);
}

PECO_API int peco_window_attention_grad(const void* q, const void* k, const void* v, const void* output,
                                        const void* grad, void* dq, void* dk, void* dv, const int64_t* strides,
                                        const int32_t* lengths, const float* row_max, const float* row_log,
                                        const void* output_rest, float* workspace, size_t workspace_floats, int batch, int q_heads, int kv_heads,
                                        int queries, int keys, int left, int right, int sinks, float scale, int d,
                                        int dtype, void* stream) {
    if (!q || !k || !v || !output || !grad || !dq || !dk || !dv || !strides || !row_max || !row_log ||
        !output_rest || !workspace ||
        !shape_ok(batch, q_heads, kv_heads, queries, keys, left, right, sinks) ||
        !(scale >= FLT_MIN && scale <= FLT_MAX) || (lengths && queries != keys))
        return kInvalidValue;
    if (d != 64 && d != 128) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16) return kUnsupportedDtype;
    if (keys > kUnbounded - 1 || queries > kUnbounded - 1 ||
        static_cast<int64_t>(queries) * (q_heads / kv_heads) > 0x7fffff00)
        return kUnsupportedShape;
    int64_t all = 0;
    for (int i = 0; i < 24; ++i) all |= strides[i];
    uintptr_t at = 0;
    for (const void* p : {q, k, v, output, grad, static_cast<const void*>(dq), static_cast<const void*>(dk),
                          static_cast<const void*>(dv), output_rest, static_cast<const void*>(workspace)})
        at |= reinterpret_cast<uintptr_t>(p);
    if (all % 8 || at % 16) return kInvalidValue;
    GradArgs A = sizes_of(batch, q_heads, kv_heads, queries, keys, left, right, sinks, d);
    const GradLayout l = grad_layout(A, d, dtype);
    if (workspace_floats < static_cast<size_t>(l.floats)) return kWorkspaceTooSmall;
    A.q = static_cast<const uint16_t*>(q);
    A.k = static_cast<const uint16_t*>(k);
    A.v = static_cast<const uint16_t*>(v);
    A.out = static_cast<const uint16_t*>(output);
    A.out_rest = static_cast<const uint16_t*>(output_rest);
    A.grad = static_cast<const uint16_t*>(grad);
    A.dq = static_cast<uint16_t*>(dq);
    A.dk = static_cast<uint16_t*>(dk);
    A.dv = static_cast<uint16_t*>(dv);
    Strides* const to[8] = {&A.qs, &A.ks, &A.vs, &A.os, &A.gs, &A.dqs, &A.dks, &A.dvs};
    for (int i = 0; i < 8; ++i) *to[i] = strides_of(strides + 3 * i);
    A.lengths = lengths;
    A.row_max = row_max;
    A.row_log = row_log;
    A.scale = scale;
    A.scale_log2 = static_cast<float>(1.4426950408889634 * static_cast<double>(scale));
    A.delta = workspace;
    A.fine_log = workspace + l.fine_log;
    A.v_long = workspace + l.v_long;
    A.g_long = workspace + l.g_long;
    A.part = A.row_part = workspace + l.part;
    const bool far = std::max(A.ks.s, A.vs.s) * 2 * keys + 2 * d >= (int64_t{1} << 32);
    const auto s = static_cast<hipStream_t>(stream);
    if (dtype == kBF16) return d == 128 ? launch_type<kBF16, 128>(A, far, s) : launch_type<kBF16, 64>(A, far, s);
    return d == 128 ? launch_type<kF16, 128>(A, far, s) : launch_type<kF16, 64>(A, far, s);
}
