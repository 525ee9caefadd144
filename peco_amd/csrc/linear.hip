// Product of rows of 8-bit codes with a weight of 8-bit codes:
//   out[m, n] = (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n],
// the sums exact in 32-bit integers (|sum| <= 2^14 k < 2^31 for k < 2^17), the rest in fp32, one rounding at the end.
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

// A workgroup's tile: kTokens x kOutputs results over blocks of kBlock channels. Its wavefronts form a grid of kM x kN,
// each with kMF x kNF products of 32 x 32, and kK of them share those results, each over every kK-th step of 32
// channels of a block. kStages blocks are in LDS or on their way.
template <int kM_, int kMF_, int kN_, int kNF_, int kK_, int kBlock_, int kStages_> struct Tile {
    static constexpr int kM = kM_, kMF = kMF_, kN = kN_, kNF = kNF_, kK = kK_, kBlock = kBlock_, kStages = kStages_;
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
    static constexpr int kLds = std::max(std::max(kStages * kStageBytes, kStoreBytes), kJoinBytes);
    static_assert(kALoads * kLoadRows * kWaves == kTokens && kWLoads * kLoadRows * kWaves == kOutputs);
    static_assert(kK == 1 || (kK == kMF * kNF && kM == 1 && kN == 1));
    static_assert(kLds + 4 * (kTokens + 2 * kOutputs) <= 160 * 1024);
    // Chunk c of row r of a block lies at place c ^ swizzle(r) of the row.
    static __device__ __forceinline__ int swizzle(int row) { return row % kChunks; }
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
            for (int i = 0; i < 4; ++i) v[i] = fmaf(static_cast<float>(acc[f][4 * g + i]) * a_scale, s[i], b[i]);
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
            if (row < rows && col < columns) *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(row) * p.n + col) = v;
        }
    } else {
        for (int e = lane; e < 32 * F * 32; e += kWave) {
            const int row = e / (F * 32), col = e % (F * 32);
            const T v = *reinterpret_cast<const T*>(span + row * kPitch + col * sizeof(T));
            if (row < rows && col < columns) out[static_cast<int64_t>(row) * p.n + col] = v;
        }
    }
}

template <int OT, typename T> __global__ __launch_bounds__(T::kThreads) void product_kernel(ProductArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __align__(128) char lds[T::kLds];
    __shared__ __align__(16) float a_scale[T::kTokens], w_scale[T::kOutputs], bias[T::kOutputs];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int tile_m = blockIdx.x % p.tiles_m, tile_n = blockIdx.x / p.tiles_m;
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
    const auto load = [&](int block) {
        const uint32_t to = lds0 + (block % T::kStages) * T::kStageBytes;
        const int8_t *from_a = a + block * T::kBlock, *from_w = w + block * T::kBlock;
        const int left = p.k - block * T::kBlock;  // a chunk behind the row's end repeats the block's first
#pragma unroll
        for (int i = 0; i < T::kALoads; ++i) {
            const int row = (i * T::kWaves + wave) * T::kLoadRows + lane / T::kChunks;
            const int at = (chunk ^ T::swizzle(row)) * 16;
            dma16_off(from_a, a_off[i] - (at < left ? 0 : at), to + i * T::kWaves * 1024);
        }
#pragma unroll
        for (int i = 0; i < T::kWLoads; ++i) {
            const int row = (i * T::kWaves + wave) * T::kLoadRows + lane / T::kChunks;
            const int at = (chunk ^ T::swizzle(row)) * 16;
            dma16_off(from_w, w_off[i] - (at < left ? 0 : at), to + T::kTokens * T::kBlock + i * T::kWaves * 1024);
        }
    };
#pragma unroll
    for (int s = 0; s < T::kStages - 1; ++s)
        if (s < blocks) load(s);

    const int in_k = wave % T::kK, in_n = wave / T::kK % T::kN, in_m = wave / T::kK / T::kN;
    const int row = lane % 32, half = lane / 32;
    const char* a_row = lds + (in_m * T::kMF * 32 + row) * T::kBlock + ((half ^ T::swizzle(row)) * 16);
    const char* w_row = lds + (T::kTokens + in_n * T::kNF * 32 + row) * T::kBlock + ((half ^ T::swizzle(row)) * 16);
    const uintptr_t a_at = reinterpret_cast<uintptr_t>(a_row), w_at = reinterpret_cast<uintptr_t>(w_row);
    i32x16 acc[T::kMF][T::kNF];
#pragma unroll
    for (int j = 0; j < T::kMF; ++j)
#pragma unroll
        for (int f = 0; f < T::kNF; ++f) acc[j][f] = i32x16{};
    const auto multiply = [&](int block, auto last) {
        const int stage = (block % T::kStages) * T::kStageBytes;
        i32x4 fa[2][T::kMF], fw[2][T::kNF];
        const auto read = [&](int s, i32x4(&x)[T::kMF], i32x4(&y)[T::kNF]) {
            const int step = s * T::kK + in_k;
            const char* at_a = reinterpret_cast<const char*>((a_at + stage) ^ (step * 32));
            const char* at_w = reinterpret_cast<const char*>((w_at + stage) ^ (step * 32));
#pragma unroll
            for (int j = 0; j < T::kMF; ++j) x[j] = *reinterpret_cast<const i32x4*>(at_a + j * 32 * T::kBlock);
#pragma unroll
            for (int f = 0; f < T::kNF; ++f) y[f] = *reinterpret_cast<const i32x4*>(at_w + f * 32 * T::kBlock);
            if constexpr (last.value) {
                const i32x4 mask = chunk_mask(p.k - block * T::kBlock - step * 32 - half * 16);
#pragma unroll
                for (int j = 0; j < T::kMF; ++j) x[j] &= mask;
            }
        };
        read(0, fa[0], fw[0]);
#pragma unroll
        for (int s = 0; s < T::kSteps; ++s) {
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < T::kSteps) read(s + 1, fa[(s + 1) % 2], fw[(s + 1) % 2]);
#pragma unroll
            for (int j = 0; j < T::kMF; ++j)
#pragma unroll
                for (int f = 0; f < T::kNF; ++f)
                    acc[j][f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s % 2][f], fa[s % 2][j], acc[j][f], 0, 0, 0);
        }
    };
    // A block is there when this wavefront's loads of it and every other's have landed; the barrier also says that the
    // block before is read, whose place the next loads take.
    for (int block = 0; block + 1 < blocks; ++block) {
        if (block + T::kStages - 1 <= blocks) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::kStages - 2) * T::kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (block + T::kStages - 1 < blocks) load(block + T::kStages - 1);
        multiply(block, std::false_type{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    multiply(blocks - 1, std::true_type{});
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

using Wide = Tile<4, 2, 2, 4, 1, 128, 2>;   // 256 x 256
using Small = Tile<1, 2, 1, 2, 4, 256, 2>;  // 64 x 64

template <int OT, typename T> int launch_product(ProductArgs p, hipStream_t s) {
    p.tiles_m = static_cast<int>(ceil_div(p.m, T::kTokens));
    p.tiles_n = static_cast<int>(ceil_div(p.n, T::kOutputs));
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    if (!fits_grid(tiles, T::kThreads)) return kUnsupportedShape;
    hipLaunchKernelGGL((product_kernel<OT, T>), dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), 0, s, p);
    return hipGetLastError();
}

template <int OT> int launch_type(const ProductArgs& p, hipStream_t s) {
    const int64_t wide = ceil_div(p.m, Wide::kTokens) * ceil_div(p.n, Wide::kOutputs);
    return 2 * wide > device_compute_units() ? launch_product<OT, Wide>(p, s) : launch_product<OT, Small>(p, s);
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
    return kOk;
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

PECO_API int peco_int8_linear_rows(const void* x, const int64_t* strides, int n0, int n1, int n2, int x_dtype,
                                   const int8_t* weight, int64_t weight_pitch, const float* weight_scales,
                                   const void* bias, int bias_wide, void* output, void* workspace,
                                   size_t workspace_bytes, int channels, int outputs, int dtype, void* stream) {
    if (!x || !strides || n0 < 1 || n1 < 1 || n2 < 1 || channels < 1) return kInvalidValue;
    if (static_cast<int64_t>(n0) * n1 > 0x3fffffff || static_cast<int64_t>(n0) * n1 * n2 > 0x3fffffff) return kUnsupportedShape;
    const int rows = n0 * n1 * n2;
    if (const int bad = check_product(weight, weight_pitch, weight_scales, output, rows, channels, outputs, dtype)) return bad;
    const int64_t pitch = ceil_div(channels, 16) * 16;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return kInvalidValue;
    if (!workspace || workspace_bytes < static_cast<size_t>(rows) * (pitch + 4)) return kWorkspaceTooSmall;
    auto* codes = static_cast<int8_t*>(workspace);
    auto* scales = reinterpret_cast<float*>(codes + rows * pitch);
    const auto s = static_cast<hipStream_t>(stream);
    if (const int bad = launch_quantize_rows(x, strides, codes, pitch, scales, n0, n1, n2, channels, x_dtype, s)) return bad;
    const ProductArgs p{codes, weight, scales, weight_scales, bias, output, pitch, weight_pitch, rows, outputs, channels,
                        bias_wide, 0, 0};
    return run_product(p, dtype, s);
}
