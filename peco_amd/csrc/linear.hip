// Product of rows of 8-bit codes with a weight of 8-bit codes:
//   out[m, n] = (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n],
// the sums exact in 32-bit integers (|sum| <= 2^14 k < 2^31 for k < 2^17), the rest in fp32, one rounding at the end. The order
// of an integer sum does not matter, so every tile and split gives the same bits.
//
// Matrix units (v_mfma_i32_32x32x32_i8) fed from LDS, which direct loads fill: a block of 128 channels of the tile's rows is a
// whole line a row (blocks of 64 fetched every line twice: 2174 against 2440 TOP/s). A tile of 256 x 256 takes 128 of a lane's
// registers for its sums and 8 wavefronts; two blocks of 64 KB lie in LDS, one barrier a block. Measured: 16384 x 4096 x 4096 225
// to 233 us, 2360-2440 TOP/s (the vendor library's 8-bit product of 8192^3 reaches 2080-2100 on the same card), the matrix
// units busy 63% of the time at 1.8 GHz; without the loads 195 us, without loads and LDS reads 167-177, the loads alone
// 140: a block's loads take 2760 cycles to land, its products 2048. 7006 x 6144 x 2048 88 us: 672 tiles are 2.6 rounds (fp32
// results 104). 8000 x 3001 x 1000 40 us in bf16, 44 to 51 in fp32: 5.9 rounds of tiles of 8 blocks.
// Walking over tiles with the next tile's loads under the stores (98 against 94 us), other shapes of the 8 wavefronts, bands of
// 2 to 16 tiles, wave priorities and rows padded off powers of two gained nothing.
#include "rows.hpp"

#include <algorithm>

namespace peco {
namespace {

struct ProductArgs {
    const int8_t *a, *w;
    const float *a_scale, *w_scale;
    const void* bias;  // nullable
    void* out;         // [m, n], contiguous
    int64_t a_pitch, w_pitch;
    int m, n, k;
    int bias_wide;     // fp32, else of the output's type
    int tiles_m, tiles_n;
};

template <int OT> __device__ __forceinline__ float load_bias(const ProductArgs& p, int n) {
    if (!p.bias) return 0.0f;
    return OT == kF32 || p.bias_wide ? static_cast<const float*>(p.bias)[n] : load_elem<OT>(p.bias, n);
}

// A result in fp32, the same bits in every kernel: rounded to fp32 before the type (a mixed-precision operation would
// round once).
__device__ __forceinline__ float scaled(int32_t sum, float a_scale, float w_scale, float bias) {
    float v = fmaf(static_cast<float>(sum) * a_scale, w_scale, bias);
    asm("" : "+v"(v));
    return v;
}

// A workgroup's tile: kTokens x kOutputs results over blocks of kBlock channels. Its wavefronts form a grid of kM x kN,
// each with kMF x kNF products of 32 x 32, and kK of them share those results, each over every kK-th step of 32
// channels of a block. Two blocks are in LDS or on their way.
template <int kM_, int kMF_, int kN_, int kNF_, int kK_, int kBlock_> struct Tile {
    static constexpr int kM = kM_, kMF = kMF_, kN = kN_, kNF = kNF_, kK = kK_, kBlock = kBlock_;
    static constexpr int kTokens = kM * kMF * 32, kOutputs = kN * kNF * 32;
    static constexpr int kWaves = kM * kN * kK, kThreads = kWaves * kWave;
    static constexpr int kChunks = kBlock / 16;               // 16-byte chunks of a row of a block
    static constexpr int kLoadRows = kWave / kChunks;         // rows of one load of a wavefront
    static constexpr int kALoads = kTokens / kLoadRows / kWaves, kWLoads = kOutputs / kLoadRows / kWaves;
    static constexpr int kLoads = kALoads + kWLoads;
    static constexpr int kSteps = kBlock / 32 / kK;           // of a wavefront in a block
    static constexpr int kStageBytes = (kTokens + kOutputs) * kBlock;
    static constexpr int kPassTiles = kK == 1 ? kNF : 1;      // 32 x 32 results a wavefront stores at once, side by side
    static constexpr int kStoreBytes = kWaves * 32 * (kPassTiles * 32 * 4 + 16);
    static constexpr int kJoinBytes = kK == 1 ? 0 : kWaves * kMF * kNF * 4096;
    static constexpr int kLds = std::max(std::max(2 * kStageBytes, kStoreBytes), kJoinBytes);
    static_assert(kALoads * kLoadRows * kWaves == kTokens && kWLoads * kLoadRows * kWaves == kOutputs);
    static_assert(kK == 1 || (kK == kMF * kNF && kM == 1 && kN == 1));
    static_assert(kLds + 4 * (kTokens + 2 * kOutputs) <= 160 * 1024);
    // Chunk c of row r of a block lies at place c ^ swizzle(r) of the row.
    static __device__ __forceinline__ int swizzle(int row) { return row / kRowsA % kChunks; }
    static constexpr int kRowsA = kChunks >= 16 ? 1 : 16 / kChunks;
};

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// Masks of the bytes of a 16-byte chunk that lie before `valid`.
__device__ __forceinline__ i32x4 chunk_mask(int valid) {
    i32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int bytes = min(max(valid - 4 * i, 0), 4);
        m[i] = bytes == 4 ? -1 : (1 << (8 * bytes)) - 1;
    }
    return m;
}

// Waits until at most N loads are on their way, or for all where fewer than that were issued behind the ones needed.
template <int N> __device__ __forceinline__ void wait_loads(bool some) {
    if (N > 0 && some) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// F 32 x 32 results of 32 tokens from m0 and 32 F outputs from n0 on: scaled, turned through LDS (the wavefront's own
// span, rows of a token's outputs) and stored in whole rows. Element r of a result: token lane % 32, output
// 8 (r / 4) + 4 (lane / 32) + r % 4.
template <int OT, int F>
__device__ __forceinline__ void store_results(const ProductArgs& p, const i32x16 (&acc)[F], char* span, int m0, int n0,
                                              float a_scale, const float* w_scale, const float* bias, int lane) {
    using T = std::conditional_t<OT == kF32, float, uint16_t>;
    constexpr int kPitch = F * 32 * sizeof(T) + 16;
    const int half = lane / 32;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int n = f * 32 + 8 * g + 4 * half;
            const f32x4 s = *reinterpret_cast<const f32x4*>(w_scale + n), b = *reinterpret_cast<const f32x4*>(bias + n);
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = scaled(acc[f][4 * g + i], a_scale, s[i], b[i]);
            char* to = span + (lane % 32) * kPitch + n * sizeof(T);
            if constexpr (OT == kF32) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
            else *reinterpret_cast<u32x2*>(to) = u32x2{Mfma<OT>::pack2(v[0], v[1]), Mfma<OT>::pack2(v[2], v[3])};
        }
    const int rows = min(32, p.m - m0), columns = min(F * 32, p.n - n0);
    T* out = static_cast<T*>(p.out) + static_cast<int64_t>(m0) * p.n + n0;
    constexpr int kPer = 16 / sizeof(T), kRowLanes = F * 32 / kPer;
    if (p.n % kPer == 0) {
#pragma unroll
        for (int r = 0; r < 32; r += kWave / kRowLanes) {
            const int row = r + lane / kRowLanes, col = lane % kRowLanes * kPer;
            const u32x4 v = *reinterpret_cast<const u32x4*>(span + row * kPitch + col * sizeof(T));
            if (row < rows && col < columns) {
                u32x4* to = reinterpret_cast<u32x4*>(out + static_cast<int64_t>(row) * p.n + col);
                if constexpr (F > 1) __builtin_nontemporal_store(v, to);  // (large results would push operands out of L2)
                else *to = v;
            }
        }
    } else {
        // 16 bytes at any element, and one by one at the end of the output's rows.
        typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
        for (int r = 0; r < 32; r += kWave / kRowLanes) {
            const int row = r + lane / kRowLanes, col = lane % kRowLanes * kPer;
            const char* from = span + row * kPitch + col * sizeof(T);
            T* to = out + static_cast<int64_t>(row) * p.n + col;
            if (row >= rows) continue;
            if (col + kPer <= columns) *reinterpret_cast<any_u32x4*>(to) = *reinterpret_cast<const u32x4*>(from);
            else
                for (int i = 0; col + i < columns; ++i) to[i] = reinterpret_cast<const T*>(from)[i];
        }
    }
}

// Workgroup i runs on XCD i % 8, each with an L2 of its own: every XCD takes a run of tiles that lie together, in bands of
// kBand tiles of tokens, so that its 32 CUs share rows and weights.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_of(const ProductArgs& p, int& tile_m, int& tile_n) {
    const int tiles = p.tiles_m * p.tiles_n, per = tiles / kXcdCount, rest = tiles % kXcdCount;
    const int xcd = blockIdx.x % kXcdCount, t = xcd * per + min(xcd, rest) + static_cast<int>(blockIdx.x) / kXcdCount;
    const int band = t / (kBand * p.tiles_n), in_band = t - band * kBand * p.tiles_n;
    const int high = min(kBand, p.tiles_m - band * kBand);
    tile_m = band * kBand + in_band % high;
    tile_n = in_band / high;
}

template <int OT, typename T> __global__ __launch_bounds__(T::kThreads) void product_kernel(ProductArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __align__(128) char lds[T::kLds];
    __shared__ __align__(16) float a_scale[T::kTokens], w_scale[T::kOutputs], bias[T::kOutputs];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int tile_m, tile_n;
    tile_of(p, tile_m, tile_n);
    const int m0 = tile_m * T::kTokens, n0 = tile_n * T::kOutputs;
    for (int i = threadIdx.x; i < T::kTokens; i += T::kThreads) a_scale[i] = p.a_scale[min(m0 + i, p.m - 1)];
    for (int i = threadIdx.x; i < T::kOutputs; i += T::kThreads) {
        const int n = min(n0 + i, p.n - 1);
        w_scale[i] = p.w_scale[n];
        bias[i] = load_bias<OT>(p, n);
    }
    // Source offsets of this lane's chunks in a block, from the tile's first row (rows past the end repeat the last).
    const int chunk = lane % T::kChunks;
    uint32_t a_off[T::kALoads], w_off[T::kWLoads];
#pragma unroll
    for (int i = 0; i < T::kALoads; ++i) {
        const int row = (i * T::kWaves + wave) * T::kLoadRows + lane / T::kChunks;
        a_off[i] = static_cast<uint32_t>(min(row, p.m - 1 - m0)) * static_cast<uint32_t>(p.a_pitch) + (chunk ^ T::swizzle(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < T::kWLoads; ++i) {
        const int row = (i * T::kWaves + wave) * T::kLoadRows + lane / T::kChunks;
        w_off[i] = static_cast<uint32_t>(min(row, p.n - 1 - n0)) * static_cast<uint32_t>(p.w_pitch) + (chunk ^ T::swizzle(row)) * 16;
    }
    const int8_t *a = p.a + m0 * p.a_pitch, *w = p.w + n0 * p.w_pitch;
    const int blocks = (p.k + T::kBlock - 1) / T::kBlock;
    const uint32_t lds0 = lds_addr(lds) + wave * 1024;
    // Loads [first, last) of this wavefront's share of a block.
    const auto load = [&](int block, int first, int last) {
        const uint32_t to = lds0 + (block % 2) * T::kStageBytes;
        const int8_t *from_a = a + block * T::kBlock, *from_w = w + block * T::kBlock;
        const int left = p.k - block * T::kBlock;  // a chunk behind the row's end repeats the block's first
#pragma unroll
        for (int i = first; i < last; ++i) {
            const bool of_a = i < T::kALoads;
            const int own = of_a ? i : i - T::kALoads;
            const int row = (own * T::kWaves + wave) * T::kLoadRows + lane / T::kChunks;
            const int at = (chunk ^ T::swizzle(row)) * 16;
            dma16_off(of_a ? from_a : from_w, (of_a ? a_off[own] : w_off[own]) - (at < left ? 0 : at),
                      to + (of_a ? 0 : T::kTokens * T::kBlock) + own * T::kWaves * 1024);
        }
    };
    load(0, 0, T::kLoads);
    if (blocks > 1) load(1, 0, T::kLoads);

    const int in_k = wave % T::kK, in_n = wave / T::kK % T::kN, in_m = wave / T::kK / T::kN;
    const int row = lane % 32, half = lane / 32;
    const int a_at = (in_m * T::kMF * 32 + row) * T::kBlock + ((half ^ T::swizzle(row)) * 16);
    const int w_at = (T::kTokens + in_n * T::kNF * 32 + row) * T::kBlock + ((half ^ T::swizzle(row)) * 16);
    i32x16 acc[T::kMF][T::kNF];
#pragma unroll
    for (int j = 0; j < T::kMF; ++j)
#pragma unroll
        for (int f = 0; f < T::kNF; ++f) acc[j][f] = i32x16{};
    // The operands of one step of 32 channels: in `now` while the products use them, the next step's on their way.
    i32x4 now_a[T::kMF], now_w[T::kNF], next_a[T::kMF], next_w[T::kNF];
    const auto read = [&](int block, int s) {
        const int stage = (block % 2) * T::kStageBytes, step = (s * T::kK + in_k) * 32;
#pragma unroll
        for (int f = 0; f < T::kNF; ++f)
            next_w[f] = *reinterpret_cast<const i32x4*>(lds + stage + (w_at ^ step) + f * 32 * T::kBlock);
#pragma unroll
        for (int j = 0; j < T::kMF; ++j)
            next_a[j] = *reinterpret_cast<const i32x4*>(lds + stage + (a_at ^ step) + j * 32 * T::kBlock);
    };
    const auto advance = [&] {
#pragma unroll
        for (int f = 0; f < T::kNF; ++f) now_w[f] = next_w[f];
#pragma unroll
        for (int j = 0; j < T::kMF; ++j) now_a[j] = next_a[j];
    };
    const auto multiply = [&](int first, int last) {
#pragma unroll
        for (int i = first; i < last; ++i)
            acc[i / T::kNF][i % T::kNF] = __builtin_amdgcn_mfma_i32_32x32x32_i8(now_w[i % T::kNF], now_a[i / T::kNF],
                                                                               acc[i / T::kNF][i % T::kNF], 0, 0, 0);
    };
    constexpr int kProducts = T::kMF * T::kNF;
    // A block's multiplication. Before its last products, whose operands are in registers: its part of LDS is read by all
    // behind the barrier and takes the block after the next (kMore: there is one), and the next has landed. The
    // products cover the barrier, the first reads behind it and the issue of the loads.
    const auto run_block = [&](int block, auto more) {
#pragma unroll
        for (int s = 0; s + 1 < T::kSteps; ++s) {
            read(block, s + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(0, kProducts);
            advance();
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(block + 1, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            multiply(i, i + 1);
            if constexpr (more.value) load(block + 2, i * T::kLoads / kProducts, (i + 1) * T::kLoads / kProducts);
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
    };
    wait_loads<T::kLoads>(blocks > 1);
    __syncthreads();
    read(0, 0);
    advance();
    for (int block = 0; block + 2 < blocks; ++block) run_block(block, std::true_type{});
    if (blocks > 1) run_block(blocks - 2, std::false_type{});
#pragma unroll
    for (int s = 0; s < T::kSteps; ++s) {
        if (s + 1 < T::kSteps) read(blocks - 1, s + 1);
        const i32x4 mask = chunk_mask(p.k - (blocks - 1) * T::kBlock - (s * T::kK + in_k) * 32 - half * 16);
#pragma unroll
        for (int j = 0; j < T::kMF; ++j) now_a[j] &= mask;
        multiply(0, kProducts);
        if (s + 1 < T::kSteps) advance();
    }
    __syncthreads();
    if constexpr (T::kK == 1) {
        char* span = lds + wave * (T::kStoreBytes / T::kWaves);
#pragma unroll
        for (int j = 0; j < T::kMF; ++j) {
            const int m = (in_m * T::kMF + j) * 32, n = in_n * T::kNF * 32;
            if (m0 + m < p.m && n0 + n < p.n)
                store_results<OT, T::kNF>(p, acc[j], span, m0 + m, n0 + n, a_scale[m + row], w_scale + n, bias + n, lane);
        }
    } else {
        // Wavefront t takes result t: the others' sums of it through LDS.
        i32x16 own[1] = {};
#pragma unroll
        for (int t = 0; t < T::kK; ++t) {
            const i32x16 v = acc[t / T::kNF][t % T::kNF];
            if (t == in_k) own[0] = v;
            else {
                i32x4* to = reinterpret_cast<i32x4*>(lds) + ((t * T::kK + in_k) * 4) * kWave + lane;
#pragma unroll
                for (int g = 0; g < 4; ++g) to[g * kWave] = i32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < T::kK; ++t)
            if (t != in_k) {
                const i32x4* from = reinterpret_cast<const i32x4*>(lds) + ((in_k * T::kK + t) * 4) * kWave + lane;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const i32x4 v = from[g * kWave];
#pragma unroll
                    for (int i = 0; i < 4; ++i) own[0][4 * g + i] += v[i];
                }
            }
        __syncthreads();
        char* span = lds + wave * (T::kStoreBytes / T::kWaves);
        const int m = in_k / T::kNF * 32, n = in_k % T::kNF * 32;
        if (m0 + m < p.m && n0 + n < p.n)
            store_results<OT, 1>(p, own, span, m0 + m, n0 + n, a_scale[m + row], w_scale + n, bias + n, lane);
    }
#endif
}

using Wide = Tile<2, 4, 4, 2, 1, 128>;   // 256 x 256
using Mid = Tile<4, 1, 2, 2, 1, 128>;    // 128 x 128
using Small = Tile<1, 2, 1, 2, 4, 256>;  // 64 x 64

// Few rows: the weight is read once, by workgroups of 16 outputs whose 8 wavefronts take segments of 256 channels in turn
// straight into registers (v_mfma_i32_16x16x64_i8, T products of 16 rows each); their sums meet in LDS. With kFused the
// rows come as x (of the output's type) and every workgroup quantizes them for itself into LDS while its first part of the
// weight is on the way, which saves a launch. Measured: 1 x 8192 x 8192 13.6 us (67 MB, 4.9 TB/s), 1 x 6144 x 2048 4.0 us, 6.5
// with the rows' quantization, for which a launch of its own takes 2.8 and its gap.
constexpr int kFewWaves = 8, kFewOutputs = 16, kSegment = 256;
constexpr int kFusedCodes = 16384;  // rows x channels

struct FewRows {
    const void* x;
    RowMap from;
};

__host__ __device__ inline int fused_pitch(int channels) { return (channels + kSegment - 1) / kSegment * kSegment + 16; }

// x's rows as codes into LDS (0 behind a row's end), their scales into `scales`. Each row is taken by 8, 4, 2 or 1
// wavefronts, 8 channels a lane at a time, and read twice (the second time from the caches).
template <int XT> __device__ __forceinline__ void quantize_into_lds(const ProductArgs& p, const FewRows& in, int8_t* codes,
                                                                    float* scales, uint32_t* most) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, pitch = fused_pitch(p.k);
    const int share = p.m == 1 ? 8 : p.m == 2 ? 4 : p.m <= 4 ? 2 : 1;  // wavefronts a row
    const int part = wave % share, lanes = share * kWave;
    for (int row = wave / share; row < p.m; row += kFewWaves / share) {
        const int64_t at = in.from.at(row);
        uint32_t top = 0;
        for (int first = 0; first < p.k; first += lanes * 8) {
            Piece<XT> x[1];
            load_row<XT, false>(x, in.x, at, RowLanes{first / 8 + part * kWave + lane, lanes, p.k});
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[0].get(k)) & 0x7fffffffu);
        }
        top = combine_lanes<MaxU, kWave>(top);
        if (lane == 0) most[row * share + part] = top;
    }
    __syncthreads();
    for (int row = wave / share; row < p.m; row += kFewWaves / share) {
        const int64_t at = in.from.at(row);
        uint32_t top = most[row * share];
        for (int i = 1; i < share; ++i) top = max(top, most[row * share + i]);
        const RowScale s(top);
        for (int first = 0; first < pitch - 16; first += lanes * 8) {
            const RowLanes r{first / 8 + part * kWave + lane, lanes, p.k};
            Piece<XT> x[1];
            load_row<XT, false>(x, in.x, at, r);
            u32x2 packed{};
#pragma unroll
            for (int k = 0; k < 8; ++k) packed[k / 4] |= (s.code(x[0].get(k)) & 0xffu) << (8 * (k % 4));
            if (r.first(0) < pitch - 16) *reinterpret_cast<u32x2*>(codes + row * pitch + r.first(0)) = packed;
        }
        if (part == 0 && lane == 0) scales[row] = s.scale();
    }
    __syncthreads();
}

template <int OT, int T, bool kFused>
__global__ __launch_bounds__(kFewWaves * kWave) void few_rows_kernel(ProductArgs p, FewRows in) {
    extern __shared__ __align__(16) int8_t few_codes[];
    __shared__ __align__(16) int32_t sums[kFewWaves][T][kWave * 4];
    __shared__ float scales[T * 16];
    __shared__ uint32_t most[16];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n0 = blockIdx.x * kFewOutputs;
    const int row = lane % 16, quarter = lane / 16;
    const int8_t* w = p.w + min(n0 + row, p.n - 1) * p.w_pitch;
    const int segments = (p.k + kSegment - 1) / kSegment;
    i32x4 weight[2][4];
    const auto load = [&](int segment, i32x4(&to)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = segment * kSegment + i * 64 + quarter * 16;
            to[i] = *reinterpret_cast<const i32x4*>(w + (at < p.k ? at : 0));  // (what is behind the end meets codes 0)
        }
    };
    if (wave < segments) load(wave, weight[0]);
    if constexpr (kFused) {
        quantize_into_lds<OT>(p, in, few_codes, scales, most);
    } else {
        for (int i = threadIdx.x; i < T * 16; i += kFewWaves * kWave) scales[i] = p.a_scale[min(i, p.m - 1)];
    }
    i32x4 acc[T] = {};
    const auto multiply = [&](int segment, const i32x4(&by)[4]) {
        i32x4 a[T][4];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int token = min(t * 16 + row, p.m - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = segment * kSegment + i * 64 + quarter * 16;
                if constexpr (kFused) a[t][i] = *reinterpret_cast<const i32x4*>(few_codes + token * fused_pitch(p.k) + at);
                else a[t][i] = *reinterpret_cast<const i32x4*>(p.a + token * p.a_pitch + (at < p.k ? at : 0));
            }
        }
        if (!kFused && (segment + 1) * kSegment > p.k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const i32x4 mask = chunk_mask(p.k - (segment * kSegment + i * 64 + quarter * 16));
#pragma unroll
                for (int t = 0; t < T; ++t) a[t][i] &= mask;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < T; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(by[i], a[t][i], acc[t], 0, 0, 0);
    };
    for (int segment = wave; segment < segments; segment += 2 * kFewWaves) {
        if (segment + kFewWaves < segments) load(segment + kFewWaves, weight[1]);
        multiply(segment, weight[0]);
        if (segment + kFewWaves >= segments) break;
        if (segment + 2 * kFewWaves < segments) load(segment + 2 * kFewWaves, weight[0]);
        multiply(segment + kFewWaves, weight[1]);
    }
    // Element r of a product: row lane % 16, output 4 (lane / 16) + r.
#pragma unroll
    for (int t = 0; t < T; ++t) *reinterpret_cast<i32x4*>(&sums[wave][t][4 * lane]) = acc[t];
    __syncthreads();
    for (int e = threadIdx.x; e < T * 256; e += kFewWaves * kWave) {
        const int token = e / 16, o = e % 16, at = 4 * (token % 16 + 16 * (o / 4)) + o % 4;
        int32_t sum = 0;
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i) sum += sums[i][token / 16][at];
        const int n = n0 + o;
        if (token >= p.m || n >= p.n) continue;
        const float v = scaled(sum, scales[token], p.w_scale[n], load_bias<OT>(p, n));
        const int64_t to = static_cast<int64_t>(token) * p.n + n;
        if constexpr (OT == kF32) static_cast<float*>(p.out)[to] = v;
        else static_cast<uint16_t*>(p.out)[to] = f32_to_half<OT>(v);
    }
}

template <int OT, int T, bool kFused> int launch_few(const ProductArgs& p, const FewRows& in, hipStream_t s) {
    const int64_t blocks = ceil_div(p.n, kFewOutputs);
    if (!fits_grid(blocks, kFewWaves * kWave)) return kUnsupportedShape;
    hipLaunchKernelGGL((few_rows_kernel<OT, T, kFused>), dim3(static_cast<unsigned>(blocks)), dim3(kFewWaves * kWave),
                       kFused ? p.m * fused_pitch(p.k) : 0, s, p, in);
    return hipGetLastError();
}

template <int OT, typename T> int launch_product(ProductArgs p, hipStream_t s) {
    p.tiles_m = static_cast<int>(ceil_div(p.m, T::kTokens));
    p.tiles_n = static_cast<int>(ceil_div(p.n, T::kOutputs));
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    if (!fits_grid(tiles, T::kThreads)) return kUnsupportedShape;
    hipLaunchKernelGGL((product_kernel<OT, T>), dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), 0, s, p);
    return hipGetLastError();
}

// Up to 32 rows the weight's bytes count (32 x 4096 x 4096 7.5 us, with small tiles 9.0; 64 rows so 11.5, with those 9.2).
// Then the tile of a product. Small ones while a round of them (two workgroups a CU) holds the result: 512 x 4096 x 4096
// takes 14.4 us with them, 20.7 with middle ones, 1024 x 2048 x 2048 9.4 and 9.6, but 512 x 6144 x 2048 14.8 and 10.3. Else by
// rounds, in units of a middle tile a CU, which run one behind the other: a round of wide tiles costs as much
// as 3.2 of them, the last one 2.3 and as much of 0.9 as it fills (2048 x 2048 in the channels: 768 middle tiles 31.4 us, 192
// wide ones 27.2; 2048 x 4096 x 4096, 512 and 128, 35.9 and 41.7; 7006 x 6144 x 2048, 2640 and 672, 100 and 88).
enum class Form { kFew, kFew2, kSmall, kMid, kWide };
Form form_of(int64_t m, int64_t n) {
    if (m <= 16) return Form::kFew;
    if (m <= 32) return Form::kFew2;
    const int64_t cus = device_compute_units();
    const auto tiles = [&](int side) { return ceil_div(m, side) * ceil_div(n, side); };
    if (tiles(Small::kTokens) <= 2 * cus) return Form::kSmall;
    const double wide = static_cast<double>(tiles(Wide::kTokens)) / cus, rounds = static_cast<double>(static_cast<int64_t>(wide));
    const double rest = wide - rounds, cost = 3.2 * rounds + (rest > 0.0 ? 2.3 + 0.9 * rest : 0.0);
    return cost <= static_cast<double>(tiles(Mid::kTokens)) / cus ? Form::kWide : Form::kMid;
}

// Whether the product's launch is one (asked before the rows' launch).
bool fits_launch(int64_t m, int64_t n) {
    const auto tiles = [&](auto tile) {
        using T = decltype(tile);
        return fits_grid(ceil_div(m, T::kTokens) * ceil_div(n, T::kOutputs), T::kThreads);
    };
    switch (form_of(m, n)) {
        case Form::kFew:
        case Form::kFew2: return fits_grid(ceil_div(n, kFewOutputs), kFewWaves * kWave);
        case Form::kSmall: return tiles(Small{});
        case Form::kMid: return tiles(Mid{});
        default: return tiles(Wide{});
    }
}

template <int OT> int launch_type(const ProductArgs& p, hipStream_t s) {
    switch (form_of(p.m, p.n)) {
        case Form::kFew: return launch_few<OT, 1, false>(p, {}, s);
        case Form::kFew2: return launch_few<OT, 2, false>(p, {}, s);
        case Form::kSmall: return launch_product<OT, Small>(p, s);
        case Form::kMid: return launch_product<OT, Mid>(p, s);
        default: return launch_product<OT, Wide>(p, s);
    }
}

}  // namespace
}  // namespace peco

using namespace peco;

namespace {

int check_product(const int8_t* weight, int64_t weight_pitch, const float* weight_scales, const void* output, int rows,
                  int channels, int outputs, int dtype) {
    if (!weight || !weight_scales || !output || rows < 1 || channels < 1 || outputs < 1 || weight_pitch < 0 ||
        weight_pitch % 16 || reinterpret_cast<uintptr_t>(weight) % 16 || reinterpret_cast<uintptr_t>(output) % 16)
        return kInvalidValue;
    if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return kUnsupportedDtype;
    // Sums of 2^17 products of -128 would leave 32 bits, and a tile's offsets are 32 bits.
    if (channels >= 1 << 17 || weight_pitch > 1 << 22 || rows > 0x3fffffff || outputs > 0x3fffffff) return kUnsupportedShape;
    return fits_launch(rows, outputs) ? kOk : kUnsupportedShape;
}

int run_product(const ProductArgs& p, int dtype, hipStream_t s) {
    switch (dtype) {
        case kBF16: return launch_type<kBF16>(p, s);
        case kF16: return launch_type<kF16>(p, s);
        default: return launch_type<kF32>(p, s);
    }
}

}  // namespace

PECO_API int peco_int8_linear(const int8_t* codes, int64_t pitch, const float* scales, const int8_t* weight,
                              int64_t weight_pitch, const float* weight_scales, const void* bias, int bias_wide,
                              void* output, int rows, int channels, int outputs, int dtype, void* stream) {
    if (const int bad = check_product(weight, weight_pitch, weight_scales, output, rows, channels, outputs, dtype)) return bad;
    if (!codes || !scales || pitch < 0 || pitch % 16 || reinterpret_cast<uintptr_t>(codes) % 16) return kInvalidValue;
    if (pitch > 1 << 22) return kUnsupportedShape;
    const ProductArgs p{codes, weight, scales, weight_scales, bias, output, pitch, weight_pitch, rows, outputs, channels,
                        bias_wide, 0, 0};
    return run_product(p, dtype, static_cast<hipStream_t>(stream));
}

namespace {

// Bytes between rows of codes: whole lines for long rows (odd lengths made the loads of 1000 channels a tenth slower).
int64_t codes_pitch(int channels) { return ceil_div(channels, channels < 512 ? 16 : 128) * (channels < 512 ? 16 : 128); }

// Whether the kernel for few rows quantizes them itself.
bool quantizes_itself(int rows, int channels, int x_dtype, int dtype) {
    return rows <= 16 && x_dtype == dtype && static_cast<int64_t>(rows) * channels <= kFusedCodes;
}

}  // namespace

PECO_API size_t peco_int8_linear_rows_workspace_size(int rows, int channels, int x_dtype, int dtype) {
    if (rows < 1 || channels < 1 || channels > kMaxRowChannels || quantizes_itself(rows, channels, x_dtype, dtype)) return 0;
    return static_cast<size_t>(rows) * (codes_pitch(channels) + 4);
}

PECO_API int peco_int8_linear_rows(const void* x, const int64_t* strides, int n0, int n1, int n2, int x_dtype,
                                   const int8_t* weight, int64_t weight_pitch, const float* weight_scales,
                                   const void* bias, int bias_wide, void* output, void* workspace,
                                   size_t workspace_bytes, int channels, int outputs, int dtype, void* stream) {
    if (!x || !strides || n0 < 1 || n1 < 1 || n2 < 1 || channels < 1) return kInvalidValue;
    if (x_dtype != kBF16 && x_dtype != kF16 && x_dtype != kF32) return kUnsupportedDtype;
    if (static_cast<int64_t>(n0) * n1 > 0x3fffffff || static_cast<int64_t>(n0) * n1 * n2 > 0x3fffffff) return kUnsupportedShape;
    const int rows = n0 * n1 * n2;
    if (const int bad = check_product(weight, weight_pitch, weight_scales, output, rows, channels, outputs, dtype)) return bad;
    if (channels > kMaxRowChannels) return kUnsupportedShape;
    const auto s = static_cast<hipStream_t>(stream);
    if (quantizes_itself(rows, channels, x_dtype, dtype)) {
        const ProductArgs p{nullptr, weight, nullptr, weight_scales, bias, output, 0, weight_pitch, rows, outputs, channels,
                            bias_wide, 0, 0};
        const FewRows in{x, row_map(strides, n0, n1, n2)};
        switch (dtype) {
            case kBF16: return launch_few<kBF16, 1, true>(p, in, s);
            case kF16: return launch_few<kF16, 1, true>(p, in, s);
            default: return launch_few<kF32, 1, true>(p, in, s);
        }
    }
    if (!workspace || workspace_bytes < peco_int8_linear_rows_workspace_size(rows, channels, x_dtype, dtype))
        return kWorkspaceTooSmall;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return kInvalidValue;
    const int64_t pitch = codes_pitch(channels);
    auto* codes = static_cast<int8_t*>(workspace);
    auto* scales = reinterpret_cast<float*>(codes + rows * pitch);
    if (const int bad = launch_quantize_rows(x, strides, codes, pitch, scales, n0, n1, n2, channels, x_dtype, s)) return bad;
    const ProductArgs p{codes, weight, scales, weight_scales, bias, output, pitch, weight_pitch, rows, outputs, channels,
                        bias_wide, 0, 0};
    return run_product(p, dtype, s);
}
