// Attention with a sliding window and sinks, over tensors or over a paged cache: forward.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that query i sees (window.hpp), 0 for a query
//   that sees none.
//
// A workgroup of 4 wavefronts takes 128 rows of one key head's row stream (its `group` query heads, token by
// token) and walks the keys that any of them sees in 64-row tiles: direct loads of the next tile's K and V
// into the other LDS buffer are in flight during the products of the current one, one barrier a tile.
//   S^T = K Q^T (32x32x16 MFMA, A = K tile rows, B = Q^T in registers): lane l holds query l % 32, keys
//         8 (i / 4) + 4 (l / 32) + i % 4 of a 32-key half;
//   softmax with a running reference (near the maximum) and sum in fp32, a lane's query its own column;
//   O^T += V^T P^T (A = V tile by transpose reads, B = P^T straight from the S^T accumulators).
// Tiles that every row of a wave sees whole run without any mask; those at the edges of the window, of the
// causal triangle and of the stream take per-element comparisons, halves that no row of the wave sees are left
// out. Items of at most 64 rows pair the waves: two waves take the same 32 rows and one 32-key half of every
// tile each, and join their states at the end.
//
// Bounds: a wave's scores, softmax and second product follow one another, and the exponentials, packing and maxima take
// about as long as the two products. Two workgroups a CU (registers allow no third) cover each other's in part only:
// MFMA is busy 39 to 44% of the time, waves wait 28 to 31% of theirs. Measured with 128 channels, bf16, calls in a row:
// 24 heads of 7006 tokens in causal windows of 2026 with 256 sinks 208 us (790 TFLOP/s of the products that the mask
// leaves, the last round of workgroups included), 3 heads of 32896 tokens in windows of 8159 491 to 536 us (743 to 811
// TFLOP/s; the clock goes between 1.8 and 2.05 GHz there, 2.3 in the former). A large library product reaches 1252. No
// LDS bank conflicts. Single tokens are bound by the keys' bytes: 119056 keys of 24 heads in 260 us (1.46 GB, 5.6 TB/s).
//
// Where items leave workgroup slots empty, their key streams are cut into `splits` parts, whose unnormalised fp32
// outputs, references and sums a second launch joins.
//
// A value that a query must not see has a weight of 0, but 0 times an infinity or NaN is NaN. A workgroup whose
// sums come out other than finite takes its item again in a careful walk, which leaves such values out of the products
// of halves that are seen in part and adds them row by row where they are seen.
//
// Roundings: scores, softmax statistics and O are fp32. P is rounded to the type for the second product (the
// sum takes the rounded values, so that the weights still add up to 1), out once at the end. Weights are relative to a
// reference, a score that no other of the row exceeds by more than 2^8 in weight: 16-bit floats round as well at 2^8 as
// at 1, and O is rescaled where the reference is raised, which after the first tiles is seldom (at every new
// maximum of any of a wave's 32 rows it was in about every other half of 76, and the first size above took a tenth longer).
#include "window.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace peco {
namespace {

// How far (in powers of two of the weights) a score may lie above its row's reference before that is raised, after the
// first tiles of a walk. There the reference is the maximum: a row of few keys is mostly its largest weight, which is 1
// then and is not rounded (with the slack from the start the gradients of windows of 16 to 256 keys are off by 1.50 to
// 1.56 times what rounding them leaves, not 1.45 to 1.48).
constexpr float kSlack = 8.0f;
constexpr int kTightTiles = 4;

struct WindowArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    Strides qs, os, ks, vs;  // paged: ks.b, vs.b are the page strides, qs.b, os.b are 0
    int heads, group;        // key heads, query heads of each
    int batch, queries, keys;  // paged: sequences, all new tokens, capacity of a table row in keys
    int left, right, sinks;
    float scale_log2;
    float slack;             // of a row's reference score (unscaled)
    const int32_t* lengths;  // contiguous: nullable valid tokens [batch]; paged: tokens held [batch]
    const int32_t* offsets;  // paged: first new token of each sequence [batch + 1]
    const int32_t* table;    // paged: page of each `page` tokens [batch, table_width]
    int64_t table_stride;
    int table_width, page, pages;
    int tiles;               // row tiles per key head (paged: an upper bound)
    int splits;              // parts of every item's key stream
    int clear_tail;          // paged: rows outside every sequence are cleared
    float* part_o;           // parts' results [splits, rows, D]
    float2* part_ml;         // and [splits, rows]: reference score, sum
    // For the backward pass (all or none): reference and log2 of the sum of every row, and what the rounding of
    // its output left (output rows one after another).
    float *row_max, *row_log;
    uint16_t* out_rest;
};

// A tile of rows, and where they are.
struct Item {
    int b, kvh;
    int row0, rows;    // rows of the stream of (b, kvh)
    int first_token;   // of the sequence within q/out
    int position0;     // position of the sequence's first query
    int queries;       // queries of the sequence that take part (later rows see nothing)
    int keys;
};

enum WindowMode : int {
    kNear = 0,   // tensors whose heads' rows lie within 2^32 bytes: 32-bit offsets from the head
    kFar = 1,    // tensors of any size
    kPaged = 2,  // pages of a cache
};

// Item i. Contiguous: heads fastest (with a multiple of 8 of them every head stays on one XCD), the last row tiles,
// which see most under a causal mask, first. Paged: heads fastest, then the row tiles of the sequences in order; false
// past the last of them.
template <int kMode> __device__ __forceinline__ bool find_rows(const WindowArgs& A, int64_t i, Item& it) {
    if constexpr (kMode != kPaged) {
        const int heads = A.batch * A.heads;
        const int bh = static_cast<int>(i % heads);
        const int tile = A.tiles - 1 - static_cast<int>(i / heads);
        it.b = bh / A.heads;
        it.kvh = bh % A.heads;
        it.first_token = 0;
        it.row0 = tile * kWinRows;
        it.rows = min(kWinRows, A.queries * A.group - it.row0);
        it.queries = A.queries;
        it.keys = A.keys;
        it.position0 = A.keys - A.queries;
        if (A.lengths) it.keys = it.queries = max(0, min(A.lengths[it.b], A.keys));  // (queries == keys)
        return true;
    } else {
        it.kvh = static_cast<int>(i % A.heads);
        int tile = static_cast<int>(i / A.heads);
        const int lane = threadIdx.x % kWave;
        for (int b0 = 0; b0 < A.batch; b0 += kWave) {
            const int b = min(b0 + lane, A.batch - 1);
            const int o0 = max(0, min(A.offsets[b], A.queries)), o1 = max(0, min(A.offsets[b + 1], A.queries));
            const int n = b0 + lane < A.batch ? max(0, o1 - o0) : 0;
            const int tiles = static_cast<int>(ceil_div(static_cast<int64_t>(n) * A.group, kWinRows));
            int upto = tiles;  // tiles of the sequences up to this lane's
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const int below = __shfl_up(upto, d, kWave);
                if (lane >= d) upto += below;
            }
            const uint64_t past = __ballot(upto > tile);
            if (past) {
                const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
                it.b = b0 + at;
                it.first_token = __shfl(o0, at, kWave);
                it.queries = __shfl(n, at, kWave);
                it.row0 = (tile - __shfl(upto - tiles, at, kWave)) * kWinRows;
                it.rows = min(kWinRows, it.queries * A.group - it.row0);
                it.keys = max(0, min(A.lengths[it.b], A.keys));
                it.position0 = it.keys - it.queries;
                return true;
            }
            tile -= __shfl(upto, kWave - 1, kWave);
        }
        it.row0 = tile;  // number among the workgroups without rows
        return false;
    }
}

// Number of a query row: query head major (paged: token major).
template <int kMode>
__device__ __forceinline__ int64_t row_number(const WindowArgs& A, const Item& it, int token, int head) {
    if constexpr (kMode == kPaged) return static_cast<int64_t>(it.first_token + token) * (A.heads * A.group) + head;
    else return (static_cast<int64_t>(it.b) * (A.heads * A.group) + head) * A.queries + token;
}

template <int kMode> __device__ __forceinline__ int64_t all_rows(const WindowArgs& A) {
    return static_cast<int64_t>(kMode == kPaged ? 1 : A.batch) * A.heads * A.group * A.queries;
}

// Clears the output rows that belong to no sequence (those before the first offset and behind the last). There
// is always a workgroup without rows (A.tiles is larger than any number of row tiles); number `at` of the `n` of a
// key head clears its share.
template <int D> __device__ void clear_tail(const WindowArgs& A, int kvh, int at, int n) {
    const int o0 = max(0, min(A.offsets[0], A.queries)), o1 = max(o0, min(A.offsets[A.batch], A.queries));
    constexpr int CH = D / 8;
    const int64_t chunks = (static_cast<int64_t>(o0) + (A.queries - o1)) * A.group * CH;
    for (int64_t i = at * int64_t{256} + threadIdx.x; i < chunks; i += n * int64_t{256}) {
        const int64_t r = i / CH, t = r / A.group;
        const int64_t token = t < o0 ? t : t - o0 + o1, head = static_cast<int64_t>(kvh) * A.group + r % A.group;
        *reinterpret_cast<u16x8*>(A.out + head * A.os.h + token * A.os.s + 8 * (i % CH)) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
}

// Four values of an output row, and with `rest` what their rounding left.
template <int DT> __device__ __forceinline__ void store_output(f32x4 x, uint16_t* out, uint16_t* rest) {
    const u32x2 w{Mfma<DT>::pack2(x[0], x[1]), Mfma<DT>::pack2(x[2], x[3])};
    *reinterpret_cast<u32x2*>(out) = w;
    if (!rest) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] -= half_to_f32<DT>(static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2))));
    *reinterpret_cast<u32x2*>(rest) = u32x2{Mfma<DT>::pack2(x[0], x[1]), Mfma<DT>::pack2(x[2], x[3])};
}

template <int DT, int D, int kMode>
__global__ __launch_bounds__(256, 2) void window_forward_kernel(WindowArgs A) {
    using T = WinTile<D>;
    constexpr int S = D / 16, NB = D / 32, H = 2;
    __shared__ __align__(256) uint16_t kvs[4][T::kElems];  // K tiles, V tiles
    uint16_t(*const ks)[T::kElems] = kvs;
    uint16_t(*const vs)[T::kElems] = kvs + 2;
    static_assert(2 * kWave * (NB * 16 + 2) * sizeof(float) <= sizeof(kvs), "pair exchange exceeds the tile LDS");
    // Paged rows: offsets (bytes) of a tile's K and V rows, whether each row counts, and page numbers on their
    // way (loaded two tiles before they are used).
    constexpr int kRowLds = kMode == kPaged ? kWinTile : 1;
    __shared__ int64_t k_off[2][kRowLds], v_off[2][kRowLds];
    __shared__ uint16_t counts[4][4];  // (read during a tile, when those two tiles on are written)
    __shared__ int page_of[2][kRowLds];

    // Parts of one item are as many workgroups apart as there are items.
    const int64_t items = static_cast<int64_t>(kMode == kPaged ? 1 : A.batch) * A.heads * A.tiles;
    const int part = static_cast<int>(blockIdx.x / items);
    Item it;
    const bool found = find_rows<kMode>(A, blockIdx.x % items, it);
    if (kMode == kPaged && !found) {
        const int tile = static_cast<int>(blockIdx.x % items / A.heads);
        if (A.clear_tail && part == 0) clear_tail<D>(A, it.kvh, it.row0, A.tiles - (tile - it.row0));
        return;
    }
    const int tid = threadIdx.x, lane = tid % kWave, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    it.keys = __builtin_amdgcn_readfirstlane(it.keys);
    it.queries = __builtin_amdgcn_readfirstlane(it.queries);
    it.position0 = __builtin_amdgcn_readfirstlane(it.position0);
    it.row0 = __builtin_amdgcn_readfirstlane(it.row0);
    it.rows = __builtin_amdgcn_readfirstlane(it.rows);
    it.b = __builtin_amdgcn_readfirstlane(it.b);
    it.first_token = __builtin_amdgcn_readfirstlane(it.first_token);

    const bool split = it.rows <= 32 * H;
    const int rb = split ? wave % H : wave;
    const int hb = split ? wave / H : 0;
    const bool wave_active = rb * 32 < it.rows;
    const int lrow = it.row0 + rb * 32 + lane % 32;  // this lane's row of the stream
    const bool qvalid = rb * 32 + lane % 32 < it.rows;
    const int token = min(lrow, it.row0 + it.rows - 1) / A.group;
    const int head = it.kvh * A.group + (min(lrow, it.row0 + it.rows - 1) - token * A.group);

    u16x8 qf[S];
    {
        const int64_t bq = kMode == kPaged ? 0 : it.b;
        const uint16_t* qrow = A.q + bq * A.qs.b + head * A.qs.h + static_cast<int64_t>(it.first_token + token) * A.qs.s;
#pragma unroll
        for (int s = 0; s < S; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qrow + 16 * s + 8 * h);
    }
    // Keys of this tile of rows, and in stream rows what this lane's query and the wave's rows see.
    const int t_first = it.row0 / A.group, t_last = min((it.row0 + it.rows - 1) / A.group, it.queries - 1);
    const KeyStream stream = t_first > t_last ? KeyStream{0, 0, 0}
                                              : key_stream(it.position0 + t_first, it.position0 + t_last, it.keys,
                                                           A.left, A.right, A.sinks);
    const int L = stream.length;
    const int all_tiles = static_cast<int>(ceil_div(L, kWinTile));
    const int per = static_cast<int>(ceil_div(all_tiles, A.splits));
    const int tile0 = min(part * per, all_tiles), tile1 = min(tile0 + per, all_tiles);
    const int pos = it.position0 + token;
    const bool sees = qvalid && token < it.queries;
    const int last_r = sees ? min(min(pos + A.right, it.keys - 1) - stream.delta, L - 1) : -1;
    const int first_r = pos - A.left - stream.delta;
    // Of the wave's rows that exist: every one sees [w_first, w_last] and the sinks up to w_last; rows past
    // w_any, and between the sinks and w_from, none of them sees.
    const int w_row0 = min(it.row0 + rb * 32, it.row0 + it.rows - 1);
    const int w_row1 = min(it.row0 + rb * 32 + 31, it.row0 + it.rows - 1);
    const int w_tok0 = w_row0 / A.group, w_tok1 = w_row1 / A.group;
    const int w_last = w_tok1 < it.queries
                           ? min(min(it.position0 + w_tok0 + A.right, it.keys - 1) - stream.delta, L - 1) : -1;
    const int w_first = it.position0 + w_tok1 - A.left - stream.delta;
    const int w_any = min(min(it.position0 + w_tok1 + A.right, it.keys - 1) - stream.delta, L - 1);
    const int w_from = it.position0 + w_tok0 - A.left - stream.delta;

    // Heads' first rows.
    const uint16_t* kh = A.k + (kMode == kPaged ? 0 : it.b) * A.ks.b + it.kvh * A.ks.h;
    const uint16_t* vh = A.v + (kMode == kPaged ? 0 : it.b) * A.vs.b + it.kvh * A.vs.h;
    const int32_t* trow = kMode == kPaged ? A.table + it.b * A.table_stride : nullptr;
    auto key_of = [&](int r) { return r < stream.a1 ? r : r + stream.delta; };
    // Tile rows 16 * wave + lane % 16 are this wave's to look up (lanes 0..15).
    constexpr int kLook = kWinTile / 4;
    const int own = kLook * wave + lane % kLook;
    const bool owner = lane < kLook;
    const int l_last = max(L - 1, 0);
    auto table_entry = [&](int r) { return trow + min(key_of(min(r, l_last)) / A.page, A.table_width - 1); };
    // Publishes this wave's rows of tile t, given the row's page number.
    auto publish = [&](int t, int buf, int page) {
        const int r = t * kWinTile + own;
        const int key = key_of(min(r, l_last));  // rows past the stream repeat its last row
        const bool ok = r < L && page >= 0 && page < A.pages;  // a page that is not held: its keys are not seen
        const int64_t p = max(0, min(page, A.pages - 1)), slot = key % A.page;
        const uint64_t bits = __ballot(ok);
        if (owner) {
            k_off[buf][own] = 2 * (p * A.ks.b + slot * A.ks.s);
            v_off[buf][own] = 2 * (p * A.vs.b + slot * A.vs.s);
        }
        if (lane == 0) counts[t % 4][wave] = static_cast<uint16_t>(bits);
    };
    auto load_tile = [&](int t, int buf) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int i = 0; i < T::kLoads; ++i) {
            const int span = i * 4 + wave;
            const int r = span * T::kWaveRows + lane / T::CH, p = lane % T::CH;
            const uint32_t chunk = (p ^ T::swz(r)) * 16;
            const uint32_t kdst = lds_addr(ks[buf] + span * kWave * 8), vdst = lds_addr(vs[buf] + span * kWave * 8);
            if constexpr (kMode != kPaged) {
                const int key = key_of(min(t * kWinTile + r, l_last));
                load_row16<kMode == kFar>(kh, key, A.ks.s, chunk, kdst);
                load_row16<kMode == kFar>(vh, key, A.vs.s, chunk, vdst);
            } else {
                dma16(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(kh) + k_off[buf][r] + chunk), kdst);
                dma16(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(vh) + v_off[buf][r] + chunk), vdst);
            }
        }
#endif
    };

    f32x16 oacc[NB];
    float m_run, l_run, neg_m;
    bool wide;
    // (From the half that the wave begins with: the second half of a tile is taken by unpaired waves, whose hb is 0.)
    const WinLane<D> at = WinLane<D>(lane, kvs[0]).moved(hb * 64 * D);

    // One 32-key half (cb) of tile t in buffer buf;
    auto compute = [&](auto careful, int t, int buf, int second) __attribute__((always_inline)) {
        constexpr bool kCareful = decltype(careful)::value;
        const int kt = 2 * (buf * T::kElems + 32 * second * D), vt = kt + 4 * T::kElems;  // bytes from `at`'s tile
        const int cb = hb + second, r0 = t * kWinTile + 32 * cb;
        if (r0 > w_any || (r0 + 31 < w_from && r0 >= A.sinks)) {  // no row of the wave sees any of it
            return;
        }
        uint32_t held = 0xffffffffu;
        if constexpr (kMode == kPaged) {
            held = __builtin_amdgcn_readfirstlane(counts[t % 4][2 * cb] | static_cast<uint32_t>(counts[t % 4][2 * cb + 1]) << 16);
        }
        const bool whole = r0 + 31 <= w_last && (r0 >= w_first || r0 + 31 < A.sinks) && held == 0xffffffffu;
        f32x16 sacc{};
#pragma unroll
        for (int s = 0; s < S; ++s) sacc = Mfma<DT>::run(at.rows(kt, s), qf[s], sacc);
        read_ahead<S, S, 4>();
        __builtin_amdgcn_sched_barrier(0);
        auto seen_at = [&](int row) {  // tile half's row -> whether this lane's query sees it
            const int r = r0 + row;
            return r <= last_r && (r >= first_r || r < A.sinks) && (held >> row & 1);
        };
        if (!whole) {
            // (Element i is row 8 (i / 4) + 4 h + i % 4: the lane's 4 h is taken off the limits, the rest is uniform.)
            const int last = last_r - 4 * h, from = first_r - 4 * h, sinks = A.sinks - 4 * h;
            const uint32_t mine = held >> (4 * h);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int c = 8 * (i / 4) + i % 4, r = r0 + c;
                if (!(r <= last && (r >= from || r < sinks) && (mine >> c & 1))) sacc[i] = -INFINITY;
            }
        }
        float tmax = sacc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) tmax = fmaxf(tmax, sacc[i]);
        const float slack = t < tile0 + kTightTiles ? 0.0f : A.slack;
        if (__any(tmax > m_run + slack)) {
            tmax = fmaxf(tmax, __shfl_xor(tmax, 32, kWave));
            const float m_new = tmax > m_run + slack ? tmax : m_run;  // (by the query's own scores alone)
            const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * A.scale_log2);
            m_run = m_new;
            // (A query that has seen nothing yet keeps its reference at the lowest value; its weights are all 0.)
            neg_m = m_new == -FLT_MAX ? 0.0f : -m_new * A.scale_log2;
            wide = __any(fabsf(neg_m) > kWideScores);  // (some query of the wave's)
            l_run *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[nb][i] *= alpha;
        }
        float offset = neg_m;
        if (wide) {  // (for the queries that need it: the others' weights keep their bits)
            const bool own = fabsf(neg_m) > kWideScores;
            const float reference = own ? m_run : 0.0f;
            if (own) offset = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sacc[i] -= reference;
        }
        uint32_t pp[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i], A.scale_log2, offset));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i + 1], A.scale_log2, offset));
            pp[i / 2] = Mfma<DT>::pack2(p0, p1);
            l_run = Mfma<DT>::sum2(pp[i / 2], l_run);
        }
        if constexpr (kCareful) {
            if (!whole && rows_not_finite<DT, D>(kvs[0], vt + hb * 64 * D, lane)) {
                add_rows_seen<DT, D>(oacc, vt, pp, at, h, seen_at);
                return;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        add_rows<DT, D>(oacc, vt, pp, at);
    };

    // One walk over the tiles.
    auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) oacc[nb] = f32x16{};
        m_run = -FLT_MAX;
        l_run = neg_m = 0.0f;
        wide = false;
        if (tile0 >= tile1) return;
        if constexpr (kMode == kPaged) {
            const int p0 = *table_entry(tile0 * kWinTile + own), p1 = *table_entry((tile0 + 1) * kWinTile + own);
            if (owner) page_of[0][own] = *table_entry((tile0 + 2) * kWinTile + own);
            publish(tile0, 0, p0);
            publish(tile0 + 1, 1, p1);
            __syncthreads();
        }
        // The query rows must have arrived before the tile loads are issued: the compiler does not count those,
        // so a later wait for the rows would also wait for the tile.
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int s = 0; s < S; ++s) asm volatile("" ::"v"(qf[s]));
#endif
        load_tile(tile0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        auto step = [&](auto bufc, int t) __attribute__((always_inline)) {
            const int buf = bufc;
            if (t + 1 < tile1) load_tile(t + 1, buf ^ 1);
            if (wave_active) {
                if constexpr (decltype(careful)::value) {
#pragma unroll 1
                    for (int second = 0; second < (split ? 1 : 2); ++second) compute(careful, t, buf, second);
                } else {
                    compute(careful, t, buf, 0);
                    if (!split) compute(careful, t, buf, 1);
                }
            }
            if constexpr (kMode == kPaged) {
                // Page numbers of tile t + 3 start on their way to LDS; those of tile t + 2 and this wave's share of
                // tile t + 1 have landed.
                const int32_t* e = table_entry((t + 3) * kWinTile + own);
                if (owner) dma4(e, lds_addr(&page_of[buf ^ 1][kLook * wave]));
                asm volatile("s_waitcnt vmcnt(1)" ::: "memory");
                // (This tile's row offsets were last read a tile ago, when its loads were issued.)
                publish(t + 2, buf, page_of[buf][own]);
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        };
        if constexpr (decltype(careful)::value) {
#pragma unroll 1
            for (int t = tile0; t < tile1; ++t) step((t - tile0) & 1, t);
        } else {
            for (int t = tile0; t < tile1; t += 2) {
                step(std::integral_constant<int, 0>{}, t);
                if (t + 1 < tile1) step(std::integral_constant<int, 1>{}, t + 1);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last page numbers
    };
    walk(std::false_type{});
    if (__syncthreads_or(wave_active && !all_finite(oacc))) walk(std::true_type{});
    if (split) {
        // The wave of the second halves leaves its state in the tile LDS (free after the last barrier), the wave of
        // the first halves joins both at the larger maximum.
        float* xch = reinterpret_cast<float*>(&kvs[0][0]) + (rb * kWave + lane) * (NB * 16 + 2);
        __syncthreads();
        if (hb == 1 && wave_active) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) xch[nb * 16 + i] = oacc[nb][i];
            xch[NB * 16] = m_run;
            xch[NB * 16 + 1] = l_run;
        }
        __syncthreads();
        if (hb == 1) return;
        if (wave_active) {
            const float m1 = xch[NB * 16], m = fmaxf(m_run, m1);
            const float a0 = __builtin_amdgcn_exp2f((m_run - m) * A.scale_log2);
            const float a1 = __builtin_amdgcn_exp2f((m1 - m) * A.scale_log2);
            m_run = m;
            l_run = l_run * a0 + xch[NB * 16 + 1] * a1;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[nb][i] = oacc[nb][i] * a0 + xch[nb * 16 + i] * a1;
        }
    }
    if (!qvalid) return;
    const float l_tot = l_run + __shfl_xor(l_run, 32, kWave);
    const int64_t row_id = row_number<kMode>(A, it, token, head);
    if (A.splits > 1) {
        const int64_t at = part * all_rows<kMode>(A) + row_id;
        if (h == 0) A.part_ml[at] = float2{m_run, l_tot};
        if (l_tot == 0.0f) return;  // (the join does not read it)
        float* o = A.part_o + at * D;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(o + 32 * nb + 8 * g + 4 * h) =
                    f32x4{oacc[nb][4 * g], oacc[nb][4 * g + 1], oacc[nb][4 * g + 2], oacc[nb][4 * g + 3]};
        return;
    }
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
    if (A.row_max && h == 0) {
        A.row_max[row_id] = m_run;
        A.row_log[row_id] = l_tot == 0.0f ? INFINITY : log2f(l_tot);
    }
    uint16_t* o = A.out + (kMode == kPaged ? 0 : it.b) * A.os.b + head * A.os.h +
                  static_cast<int64_t>(it.first_token + token) * A.os.s;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x4 x{oacc[nb][4 * g], oacc[nb][4 * g + 1], oacc[nb][4 * g + 2], oacc[nb][4 * g + 3]};
            store_output<DT>(x * inv, o + 32 * nb + 8 * g + 4 * h,
                             A.row_max ? A.out_rest + row_id * D + 32 * nb + 8 * g + 4 * h : nullptr);
        }
}

// Joins the parts of every row: out = sum_s 2^((m_s - M) scale) O_s / sum_s 2^((m_s - M) scale) l_s, in a fixed
// order. D / 4 lanes a row; kWide: one row a workgroup, whose lane groups take the parts in turn and are joined in LDS
// (a call with many parts has few rows, and one lane group would wait for one part after another).
template <int DT, int D, int kMode, bool kWide>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs A) {
    constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ f32x4 group_o[kWide ? kGroups : 1][kLanes];
    __shared__ float2 group_ml[kWide ? kGroups : 1];
    const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, c = 4 * lane, hq = A.heads * A.group;
    const int64_t rows_all = all_rows<kMode>(A);
    const int64_t row = kWide ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kGroups + group;
    if (row >= rows_all) return;
    int64_t b = 0, head, token;
    if constexpr (kMode == kPaged) {
        token = row / hq;
        head = row % hq;
        const int o0 = max(0, min(A.offsets[0], A.queries)), o1 = min(A.offsets[A.batch], A.queries);
        if (token < o0 || token >= o1) return;  // of no sequence: no parts were written
    } else {
        token = row % A.queries;
        head = row / A.queries % hq;
        b = row / A.queries / hq;
    }
    float m = -FLT_MAX, l = 0.0f;
    f32x4 o{};
    const int first = kWide ? group : 0, step = kWide ? kGroups : 1;
    for (int s = first; s < A.splits; s += step) m = fmaxf(m, A.part_ml[s * rows_all + row].x);
    for (int s = first; s < A.splits; s += step) {
        const float2 ml = A.part_ml[s * rows_all + row];
        if (ml.y == 0.0f) continue;
        const float w = __builtin_amdgcn_exp2f((ml.x - m) * A.scale_log2);
        const f32x4 part = *reinterpret_cast<const f32x4*>(A.part_o + (s * rows_all + row) * D + c);
        l += w * ml.y;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] += w * part[k];
    }
    if constexpr (kWide) {
        group_o[group][lane] = o;
        if (lane == 0) group_ml[group] = float2{m, l};
        __syncthreads();
        if (group) return;
        const float own = m;
#pragma unroll
        for (int i = 1; i < kGroups; ++i) m = fmaxf(m, group_ml[i].x);
        const float w0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((own - m) * A.scale_log2);
        l *= w0;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = l == 0.0f ? 0.0f : o[k] * w0;
        for (int i = 1; i < kGroups; ++i) {
            const float2 ml = group_ml[i];
            if (ml.y == 0.0f) continue;
            const float w = __builtin_amdgcn_exp2f((ml.x - m) * A.scale_log2);
            l += w * ml.y;
            const f32x4 x = group_o[i][lane];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] += w * x[k];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (A.row_max && c == 0) {
        A.row_max[row] = m;
        A.row_log[row] = l == 0.0f ? INFINITY : log2f(l);
    }
    uint16_t* dst = A.out + b * A.os.b + head * A.os.h + token * A.os.s + c;
    store_output<DT>(o * inv, dst, A.row_max ? A.out_rest + row * D + c : nullptr);
}

constexpr int kWideParts = 8;  // parts from which the join takes a workgroup a row

template <int DT, int D, int kMode> int launch_join(const WindowArgs& A, int64_t rows, hipStream_t s) {
    constexpr int kGroups = 256 / (D / 4);
    if (A.splits >= kWideParts)
        hipLaunchKernelGGL((window_join_kernel<DT, D, kMode, true>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, A);
    else
        hipLaunchKernelGGL((window_join_kernel<DT, D, kMode, false>), dim3(static_cast<unsigned>(ceil_div(rows, kGroups))),
                           dim3(256), 0, s, A);
    return hipGetLastError();
}

template <int DT, int D, int kMode> int launch_mode(const WindowArgs& A, hipStream_t s) {
    const int64_t rows = (kMode == kPaged ? int64_t{1} : int64_t{A.batch}) * A.heads * A.group * A.queries;
    const int64_t blocks = (kMode == kPaged ? int64_t{1} : int64_t{A.batch}) * A.heads * A.tiles * A.splits;
    const dim3 grid(static_cast<unsigned>(blocks));
    hipLaunchKernelGGL((window_forward_kernel<DT, D, kMode>), grid, dim3(256), 0, s, A);
    const int status = hipGetLastError();
    if (status || A.splits == 1) return status;
    return launch_join<DT, D, kMode == kFar ? kNear : kMode>(A, rows, s);
}

template <int DT, int D> int launch_window(const WindowArgs& A, WindowMode mode, hipStream_t s) {
    switch (mode) {
        case kNear: return launch_mode<DT, D, kNear>(A, s);
        case kFar: return launch_mode<DT, D, kFar>(A, s);
        default: return launch_mode<DT, D, kPaged>(A, s);
    }
}

int launch(const WindowArgs& A, WindowMode mode, int d, int dtype, hipStream_t s) {
    if (dtype == kBF16) return d == 128 ? launch_window<kBF16, 128>(A, mode, s) : launch_window<kBF16, 64>(A, mode, s);
    return d == 128 ? launch_window<kF16, 128>(A, mode, s) : launch_window<kF16, 64>(A, mode, s);
}

struct Shape {
    int64_t tiles, rows, blocks;  // row tiles of a key head, query rows, workgroups
    int splits;
};

// Whether the forward's and the join's launches are ones (the rows' number has to be an int as well).
bool launchable(const Shape& s, int d) {
    const int64_t join = s.splits == 1 ? 0 : s.splits >= kWideParts ? s.rows : ceil_div(s.rows, 256 / (d / 4));
    return s.rows <= 0x7fffffff && fits_grid(std::max(s.blocks, join), 256);
}

// Into how many parts (of at least kPartTiles tiles) the key streams are cut.
// Items of a few rows (single tokens) are bound by what they read: about four workgroups a slot (two slots a CU) keep
// the reads even where sequences differ in length. Measured, 128 channels: 32 x 8 heads of one token over up to 7006
// keys 176 us uncut, 106 in 8 parts and 5 for the join; one token over 119056 keys, 24 heads, 298 us in 12 parts, 359
// in 21 (one even round, whose last workgroups read alone), 271 in 64 and 13 for the join. (97 and 260 us since.)
// Other items are bound by their products (cut_parts).
constexpr int kFewRows = 32;
// `heads` key heads of `tiles` row tiles, `items` of them with rows, which hold `rows` in all.
Shape shape_of(int64_t heads, int64_t tiles, int64_t items, int64_t seen_keys, int64_t rows, int d) {
    Shape best{tiles, rows, 0, 1};
    if (rows <= items * kFewRows)
        best.splits = static_cast<int>(std::min(most_parts(seen_keys), ceil_div(8 * int64_t{device_compute_units()}, items)));
    else best.splits = cut_parts(items, seen_keys, rows, d);
    best.blocks = heads * tiles * best.splits;
    return best;
}

Shape window_shape(int batch, int q_heads, int kv_heads, int queries, int keys, int left, int right, int sinks, int d) {
    const int group = q_heads / kv_heads;
    const int64_t tiles = ceil_div(static_cast<int64_t>(queries) * group, kWinRows), heads = int64_t{batch} * kv_heads;
    const int64_t tokens = std::min<int64_t>(queries, kWinRows / group + 1);
    return shape_of(heads, tiles, heads * tiles, seen_keys(keys, tokens, left, right, sinks), heads * group * queries, d);
}

// Row tiles of a ragged batch: each sequence has at most one that is not full; one more, so that some
// workgroup always finds no rows and clears those outside every sequence.
Shape paged_shape(int batch, int q_heads, int kv_heads, int tokens, int64_t capacity, int left, int sinks, int d) {
    const int group = q_heads / kv_heads;
    const int64_t full = static_cast<int64_t>(tokens) * group / kWinRows, tiles = full + batch + 1;
    const int64_t some = std::min<int64_t>(tokens, kWinRows / group + 1);
    return shape_of(kv_heads, tiles, (tiles - 1) * kv_heads, seen_keys(capacity, some, left, 0, sinks),
                 static_cast<int64_t>(tokens) * q_heads, d);
}

size_t workspace_floats(const Shape& s, int d) {
    return s.splits > 1 ? static_cast<size_t>(s.splits) * s.rows * (d + 2) : 0;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned(const Strides& s) { return (s.b | s.h | s.s) % 8 == 0; }

bool mask_ok(int left, int right, int sinks) {
    return left >= -1 && right >= -1 && sinks >= 0 && left <= kUnbounded && right <= kUnbounded && sinks <= kUnbounded;
}
// (A negative scale would turn the running maximum into a minimum, 0 times a masked score is NaN.)
bool scale_ok(float scale) { return scale >= FLT_MIN && scale <= FLT_MAX; }
int unbounded(int n) { return n < 0 ? kUnbounded : n; }

void set_scale(WindowArgs& A, float scale) {
    A.scale_log2 = static_cast<float>(1.4426950408889634 * static_cast<double>(scale));
    A.slack = std::min(kSlack / A.scale_log2, 0x1p100f);  // (added to the lowest float it must stay below every score)
}

void set_parts(WindowArgs& A, const Shape& s, float* workspace, int d) {
    A.splits = s.splits;
    A.tiles = static_cast<int>(s.tiles);
    A.part_o = workspace;
    A.part_ml = reinterpret_cast<float2*>(workspace + static_cast<int64_t>(s.splits) * s.rows * d);
}

Strides strides_of(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

}  // namespace
}  // namespace peco

using namespace peco;

PECO_API size_t peco_window_attention_workspace_size(int batch, int q_heads, int kv_heads, int queries, int keys,
                                                     int left, int right, int sinks, int d) {
    if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || queries < 1 || keys < 0) return 0;
    return workspace_floats(window_shape(batch, q_heads, kv_heads, queries, keys, left, right, sinks, d), d);
}

PECO_API int peco_window_attention(const void* q, const void* k, const void* v, void* output, const int64_t* strides,
                                   const int32_t* lengths, float* row_max, float* row_log, void* output_rest,
                                   float* workspace, size_t workspace_floats_given, int batch, int q_heads, int kv_heads, int queries,
                                   int keys, int left, int right, int sinks, float scale, int d, int dtype,
                                   void* stream) {
    if (!q || !k || !v || !output || !strides || !row_max != !row_log || !row_max != !output_rest || batch < 1 || kv_heads < 1 ||
        q_heads < kv_heads || q_heads % kv_heads || queries < 1 || keys < 1 || !mask_ok(left, right, sinks) ||
        !scale_ok(scale) || (lengths && queries != keys))
        return kInvalidValue;
    if (d != 64 && d != 128) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16) return kUnsupportedDtype;
    if (keys > kUnbounded - 1 || queries > kUnbounded - 1 ||
        static_cast<int64_t>(queries) * (q_heads / kv_heads) > 0x7fffff00)
        return kUnsupportedShape;
    WindowArgs A{};
    A.qs = strides_of(strides);
    A.ks = strides_of(strides + 3);
    A.vs = strides_of(strides + 6);
    A.os = strides_of(strides + 9);
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(output) || !aligned(A.qs) || !aligned(A.ks) ||
        !aligned(A.vs) || !aligned(A.os))
        return kInvalidValue;
    A.q = static_cast<const uint16_t*>(q);
    A.k = static_cast<const uint16_t*>(k);
    A.v = static_cast<const uint16_t*>(v);
    A.out = static_cast<uint16_t*>(output);
    A.heads = kv_heads;
    A.group = q_heads / kv_heads;
    A.batch = batch;
    A.queries = queries;
    A.keys = keys;
    A.left = unbounded(left);
    A.right = unbounded(right);
    A.sinks = sinks;
    set_scale(A, scale);
    A.lengths = lengths;
    A.row_max = row_max;
    A.row_log = row_log;
    A.out_rest = static_cast<uint16_t*>(output_rest);
    if (!aligned(output_rest)) return kInvalidValue;
    const Shape shape = window_shape(batch, q_heads, kv_heads, queries, keys, left, right, sinks, d);
    if (!launchable(shape, d)) return kUnsupportedShape;
    if (workspace_floats(shape, d) > workspace_floats_given) return kWorkspaceTooSmall;
    if (workspace_floats(shape, d) && (!workspace || !aligned(workspace))) return kInvalidValue;
    set_parts(A, shape, workspace, d);
    const int64_t reach = std::max(A.ks.s, A.vs.s) * 2 * keys + 2 * d;
    return launch(A, reach < (int64_t{1} << 32) ? kNear : kFar, d, dtype, static_cast<hipStream_t>(stream));
}

PECO_API size_t peco_paged_attention_workspace_size(int batch, int q_heads, int kv_heads, int tokens, int table_width,
                                                    int page, int left, int sinks, int d) {
    if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || tokens < 1 || table_width < 1 || page < 1)
        return 0;
    const int64_t capacity = static_cast<int64_t>(table_width) * page;
    return workspace_floats(paged_shape(batch, q_heads, kv_heads, tokens, capacity, left, sinks, d), d);
}

PECO_API int peco_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* output,
                                  const int64_t* strides, const int32_t* page_table, int64_t table_stride,
                                  const int32_t* offsets, const int32_t* lengths, int clear_tail, float* workspace,
                                  size_t workspace_floats_given, int batch, int q_heads, int kv_heads, int tokens,
                                  int pages, int page, int table_width, int left, int sinks, float scale, int d,
                                  int dtype, void* stream) {
    if (!q || !k_pages || !v_pages || !output || !strides || !page_table || !offsets || !lengths || batch < 1 ||
        kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || tokens < 1 || pages < 1 || page < 1 ||
        table_width < 1 || table_stride < 0 || !mask_ok(left, 0, sinks) || !scale_ok(scale))
        return kInvalidValue;
    if (d != 64 && d != 128) return kUnsupportedShape;
    if (dtype != kBF16 && dtype != kF16) return kUnsupportedDtype;
    const int64_t capacity = static_cast<int64_t>(table_width) * page;
    if (capacity > kUnbounded - 1 || tokens > kUnbounded - 1 ||
        static_cast<int64_t>(tokens) * (q_heads / kv_heads) > 0x7fffff00)
        return kUnsupportedShape;
    WindowArgs A{};
    A.qs = Strides{0, strides[0], strides[1]};
    A.ks = strides_of(strides + 2);
    A.vs = strides_of(strides + 5);
    A.os = Strides{0, strides[8], strides[9]};
    if (!aligned(q) || !aligned(k_pages) || !aligned(v_pages) || !aligned(output) || !aligned(A.qs) || !aligned(A.ks) ||
        !aligned(A.vs) || !aligned(A.os))
        return kInvalidValue;
    A.q = static_cast<const uint16_t*>(q);
    A.k = static_cast<const uint16_t*>(k_pages);
    A.v = static_cast<const uint16_t*>(v_pages);
    A.out = static_cast<uint16_t*>(output);
    A.heads = kv_heads;
    A.group = q_heads / kv_heads;
    A.batch = batch;
    A.queries = tokens;
    A.keys = static_cast<int>(capacity);
    A.left = unbounded(left);
    A.right = 0;
    A.sinks = sinks;
    set_scale(A, scale);
    A.lengths = lengths;
    A.offsets = offsets;
    A.table = page_table;
    A.table_stride = table_stride;
    A.table_width = table_width;
    A.page = page;
    A.pages = pages;
    A.clear_tail = clear_tail;
    const Shape shape = paged_shape(batch, q_heads, kv_heads, tokens, capacity, left, sinks, d);
    if (!launchable(shape, d)) return kUnsupportedShape;
    if (workspace_floats(shape, d) > workspace_floats_given) return kWorkspaceTooSmall;
    if (workspace_floats(shape, d) && (!workspace || !aligned(workspace))) return kInvalidValue;
    set_parts(A, shape, workspace, d);
    return launch(A, kPaged, d, dtype, static_cast<hipStream_t>(stream));
}
