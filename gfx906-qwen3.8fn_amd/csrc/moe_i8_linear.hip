// Matrices of int8 codes with one fp32 scale per output channel
// (moe_i8_linear_*) and the quantiser of their activations.
#include "moe_ffn.h"
#include "moe_i8.hpp"

#include <algorithm>
#include <new>

namespace moe {
namespace {

// --------------------------------------------------------------- layout ---
// One thread per 16-byte piece of the blocks that a matrix' rows fill.
__global__ __launch_bounds__(256) void k_i8_repack(const int8_t *__restrict__ codes, uint4 *__restrict__ blocks, int rows,
                                                   int cols, int chunks, size_t pieces, int part) {
    const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int lane = static_cast<int>(i & 63), tile = static_cast<int>(i >> 6) & 3, per = i8_rows(rows) / kI8Block;
    const size_t block = i >> 8, chunk = block % chunks, at = block / chunks;   // at: 64 rows, over all matrices
    const size_t matrix = at / per;
    const int r = lane & 15, in = part == kI8Whole ? (tile >> 1) * 32 + (r >> 2) * 8 + (tile & 1) * 4 + (r & 3) : tile * 16 + r;
    const int row = static_cast<int>(at % per) * kI8Block + in;
    const int col = static_cast<int>(chunk) * kI8Chunk + (lane >> 4) * 16;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows && col < cols) __builtin_memcpy(&v, codes + (matrix * rows + row) * cols + col, 16);
    const int t = part == kI8Whole ? tile : 2 * tile + part;   // of a pair's eight
    const size_t to = part == kI8Whole ? at : 2 * at + (t >> 2);
    blocks[((to * chunks + chunk) * 4 + (t & 3)) * 64 + lane] = v;
}

// ------------------------------------------------------------- quantiser ---
template<int T, int L, int V>
__global__ __launch_bounds__(256) void k_quantize_i8(I8Rows r) { quantize_rows<T, L, V>(r, blockIdx.x); }

}  // namespace

hipError_t launch_i8_repack(const int8_t *codes, uint8_t *blocks, size_t matrices, int rows, int cols, int part,
                            hipStream_t s) {
    const int chunks = i8_chunks(cols);
    // A grid holds fewer than 2^32 threads: at most 2^30 pieces a launch.
    const size_t each = static_cast<size_t>(i8_rows(rows)) / kI8Block * chunks * 256;
    const size_t at_once = std::max<size_t>(1, (size_t{1} << 30) / each);
    for (size_t first = 0; first < matrices; first += at_once) {
        const size_t n = std::min(at_once, matrices - first), pieces = n * each;
        k_i8_repack<<<dim3(static_cast<unsigned>((pieces + 255) / 256)), dim3(256), 0, s>>>(
            codes + first * rows * cols, reinterpret_cast<uint4 *>(blocks + first * each * 16 * (part == kI8Whole ? 1 : 2)), rows,
            cols, chunks, pieces, part);
    }
    return hipGetLastError();
}

hipError_t launch_quantize_i8(const I8Rows &r, int type, hipStream_t s) {
    with_quantizer(type, r.width, [&](auto t, auto l, auto v) {
        k_quantize_i8<t, l, v><<<dim3(quantize_blocks(r.rows, l)), dim3(256), 0, s>>>(r);
    });
    return hipGetLastError();
}

namespace {

// Workgroup i runs on XCD i % 8, whose L2 the others do not see: each XCD takes a
// run of the output's tiles, in columns of eight tiles of the matrix.
template<int WR, int WC, int TM, int TN, int S, int KS, int Y>
__global__ __launch_bounds__(64 * WR * WC) void k_i8_gemm(I8Args a) {
    using Stream = I8Stream<WR, WC, TM, TN, S, KS, kStoreRows, Y, false>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Stream::Lds];
    const int tn = (a.N + Stream::BN - 1) / Stream::BN, total = a.tiles_m * tn, each = (total + 7) / 8;
    const int xcd = static_cast<int>(blockIdx.x & 7);
    const auto fetch = [&](int i) {
        constexpr int P = 8;
        const int panel = i / (P * tn), r = i - panel * P * tn, p = min(P, a.tiles_m - panel * P);
        const int m = panel * P + r % p, n = r / p;
        return I8Item{0, m * Stream::BM, n * Stream::BN, min(a.N - n * Stream::BN, Stream::BN), tn == 1};
    };
    Stream g(a, lds);
    g.run(xcd * each + static_cast<int>(blockIdx.x >> 3), static_cast<int>(gridDim.x >> 3), min(total, (xcd + 1) * each), fetch,
          [&](const I8Item &it, const float *params, const i32x4 (&acc)[TM][TN]) { g.store_rows(it, params, acc); });
}

// Few rows of x (at most 16): a workgroup takes 16 results of each, one tile of every
// chunk, and its waves share out the chunks (wave w: chunks w, w + W, ..), the
// matrix straight from memory into registers.  IN: x's type, quantised here by
// every workgroup while its first tiles are on their way; or kCodes.  What bounds
// it: the launch and one trip to memory, then HBM.
struct I8FewArgs {
    const uint8_t *blocks;
    const float *sw;
    const void *x;        // rows of IN, x_stride elements apart, or codes
    int64_t x_stride;
    const float *sx;      // kCodes
    void *y;
    int64_t y_stride;
    int y_type, M, N, K, chunks;
    int *error;
};
inline constexpr int kFewRows = 16, kFewWaves = 8, kFewVectors = 4;   // vectors of 8 that a thread quantises
template<int IN, int Y>
__global__ __launch_bounds__(64 * kFewWaves) void k_i8_few(I8FewArgs a) {
    constexpr bool Quantize = IN != kCodes;
    constexpr int U = 4, T = 64 * kFewWaves;   // chunks of a wave in flight
    __shared__ i32x4 red[kFewWaves][64];
    __shared__ uint32_t most[kFewRows];
    extern __shared__ __attribute__((aligned(16))) uint8_t codes[];   // Quantize: [piece of 16][row][16]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x;
    const uint8_t *w = a.blocks + static_cast<size_t>(tile >> 2) * a.chunks * kI8BlockBytes + (tile & 3) * 1024 + lane * 16;
    uint4 f[U];
    const auto load = [&](int c0) {
        const auto one = [&](int u) { f[u] = load_once(w + static_cast<size_t>(c0 + u * kFewWaves) * kI8BlockBytes); };
        // All at once, without a branch between them; where there are fewer, no others
        // in their place (8192 of 2560 at 8 rows 9.4 -> 8.7 us).
        if (c0 + (U - 1) * kFewWaves < a.chunks) {
#pragma unroll
            for (int u = 0; u < U; ++u) one(u);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * kFewWaves < a.chunks) one(u);
        }
    };
    load(wave);
    if constexpr (Quantize) {
        // A thread's vectors stay in registers between their row's maximum and the codes.
        const int per = a.K / 8;
        if (threadIdx.x < kFewRows) most[threadIdx.x] = 0;
        Raw8 raw[kFewVectors];
#pragma unroll
        for (int j = 0; j < kFewVectors; ++j) {
            const int i = j * T + threadIdx.x, n = i / per;
            raw[j] = load8_any<IN>(a.x, static_cast<size_t>(n) * a.x_stride + i % per * 8, n < a.N ? 8 : 0);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kFewVectors; ++j) {
            const int n = (j * T + threadIdx.x) / per;
            float v[8];
            unpack8<IN>(raw[j], v);
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) m = max(m, magnitude(v[q]));
            // Four neighbouring threads have one row's vectors (K is a multiple of 32).
            m = max(m, static_cast<uint32_t>(lane_xor<1>(static_cast<int>(m))));
            m = max(m, static_cast<uint32_t>(lane_xor<2>(static_cast<int>(m))));
            if ((threadIdx.x & 3) == 0 && n < a.N) atomicMax(&most[n], m);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kFewVectors; ++j) {
            const int i = j * T + threadIdx.x, n = i / per, k = i % per;
            if (n >= a.N) break;
            float v[8];
            unpack8<IN>(raw[j], v);
            *reinterpret_cast<uint2 *>(codes + (static_cast<size_t>(k >> 1) * a.N + n) * 16 + (k & 1) * 8) = quantize8_i8(v, row_scale(most[n]));
        }
        if (a.K % kI8Chunk) {   // the last chunk's second half meets zeros of the matrix, as whole numbers
            for (int i = threadIdx.x; i < a.N * 8; i += T)
                reinterpret_cast<uint32_t *>(codes + static_cast<size_t>(a.K / 16) * a.N * 16)[i] = 0;
        }
        __syncthreads();
    }
    const int n = min(lane & 15, a.N - 1);
    const int8_t *rows = static_cast<const int8_t *>(a.x) + (Quantize ? 0 : static_cast<size_t>(n) * a.x_stride + (lane >> 4) * 16);
    i32x4 acc = {0, 0, 0, 0};
    for (int c0 = wave; c0 < a.chunks; c0 += kFewWaves * U) {
        if (c0 != wave) load(c0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * kFewWaves;
            if (c >= a.chunks) break;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (Quantize) x = *reinterpret_cast<const uint4 *>(codes + (static_cast<size_t>(c * 4 + (lane >> 4)) * a.N + n) * 16);
            else if (c * kI8Chunk + (lane >> 4) * 16 < a.K) x = *reinterpret_cast<const uint4 *>(rows + c * kI8Chunk);
            acc = i8_dot(f[u], x, acc);
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int j = 1; j < kFewWaves; ++j) acc += red[j][lane];
    const int row = lane & 15;
    if (row >= a.N) return;
    float sx;
    if constexpr (Quantize) {
        const GroupScale s = row_scale(most[row]);
        sx = s.s;
        if (s.bad && blockIdx.x == 0 && lane < 16) atomicOr(a.error, 1);
    } else {
        sx = a.sx[row];
    }
    const int m = (tile >> 1) * 32 + (lane >> 4) * 8 + (tile & 1) * 4;
    if (m >= a.M) return;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = static_cast<float>(acc[q]) * (sx * a.sw[m + q]);   // there up to i8_rows(M)
    const size_t at = static_cast<size_t>(row) * a.y_stride + m;
    if (m + 3 < a.M) {
        store4<Y>(a.y, at, v);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (m + q < a.M) store1<Y>(a.y, at + q, v[q]);
    }
}

template<int IN>
hipError_t launch_few(const I8FewArgs &a, hipStream_t s) {
    const dim3 block(64 * kFewWaves);
    const size_t lds = IN == kCodes ? 0 : static_cast<size_t>(a.N) * a.chunks * kI8Chunk;
    const dim3 blocks(static_cast<unsigned>(i8_rows(a.M) / 16));
    if (a.y_type == kF32) k_i8_few<IN, kF32><<<blocks, block, lds, s>>>(a);
    else if (a.y_type == kBF16) k_i8_few<IN, kBF16><<<blocks, block, lds, s>>>(a);
    else k_i8_few<IN, kF16><<<blocks, block, lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_i8_linear {
    int input = 0, output = 0, max_columns = 0, device = 0;
    uint8_t *mem = nullptr;   // blocks, scales
    const float *scales = nullptr;
    int8_t *ws = nullptr;     // rows of `pitch` codes, then their scales
    int64_t pitch = 0;
};

namespace {

constexpr int kInvalid = hipErrorInvalidValue;

bool aligned(const void *p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
bool is_type(int t) { return t == MOE_F32 || t == MOE_BF16 || t == MOE_F16; }
// Rows of `width` elements of `type` at p, `stride` elements apart.
bool valid_rows(const void *p, int type, int64_t stride, int width) {
    return is_type(type) && aligned(p, moe::elem_bytes(type)) && stride >= width && stride <= (int64_t{1} << 40);
}

void release(moe_i8_linear *L) {
    if (L->mem) (void)hipFree(L->mem);
    if (L->ws) (void)hipFree(L->ws);
    delete L;
}

inline constexpr int kFewElements = moe::kFewVectors * 64 * moe::kFewWaves * 8;   // of x, quantised inside the product
inline constexpr int kFewOutputs = 16 * 4 * 256;

template<int WR, int WC, int TM, int TN, int S, int KS>
int launch_gemm(moe::I8Args a, int y_type, hipStream_t s) {
    using Stream = moe::I8Stream<WR, WC, TM, TN, S, KS, moe::kStoreRows, moe::kF32, false>;   // sizes are those of any type
    a.tiles_m = (a.M + Stream::BM - 1) / Stream::BM;
    const size_t total = static_cast<size_t>(a.tiles_m) * ((a.N + Stream::BN - 1) / Stream::BN);
    const size_t resident = 256 * std::min(4, 160 * 1024 / Stream::Lds);
    const dim3 grid(static_cast<unsigned>(std::min((total + 7) / 8 * 8, resident))), block(64 * Stream::W);
    if (y_type == MOE_F32) moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kF32><<<grid, block, 0, s>>>(a);
    else if (y_type == MOE_BF16) moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kBF16><<<grid, block, 0, s>>>(a);
    else moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kF16><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

moe::I8FewArgs few_args(const moe_i8_linear *L, const void *x, int64_t x_stride, const float *sx, int columns, void *y, int y_type,
                        int64_t y_stride, int *error) {
    return moe::I8FewArgs{L->mem, L->scales, x, x_stride, sx, y, y_stride, y_type, L->output, columns, L->input,
                          moe::i8_chunks(L->input), error};
}

// The product for quantised rows.  The output tile grows with the number of tiles, by
// how they fill the 256 CUs, and is no wider than the rows of x.  us for forward (MI355X,
// launches in a row), bf16, tiles of 64 x 16 / 64 x 32 in stages of four chunks / of two /
// 64 x 64 / 64 x 128 / 128 x 128 / 256 x 256:
//         2048 x 2048 at   40:   5.6 /  5.9 /  6.5 /   -  /   -  /   -  /   -
//                         130:   8.9 /  6.0 /  6.6 /  7.0 /   -  /   -  /   -
//                         300:    -  /  9.8 /  8.2 /  7.1 /   -  /   -  /   -
//                         333:  10.5 /   -  /  8.1 /  7.1 /  8.8 / 12.0 / 27.2
//                        1032:  25.9 /   -  / 14.4 / 13.3 / 15.0 / 12.3 / 26.8
//                        2500:    -  /   -  /   -  / 22.6 / 20.9 / 19.0 /   -
//                        4096:  86.0 /   -  / 39.8 / 34.1 / 27.8 / 22.4 / 30.4
//         2560 x 2560 at  700:    -  /   -  / 14.8 / 12.0 / 10.7 / 14.5 /   -
//         2048 of 8192, 200:      -  / 14.8 / 17.8 / 16.8 /   -  /   -  /   -
//                       600:      -  /   -  / 28.7 / 28.9 / 24.7 / 35.6 /   -   (fp32)
//         8192 x 8192 at   20:  14.4 / 17.9 / 26.3 / 27.0 /   -  /   -  /   -
//                          64:  21.1 /   -  / 17.6 / 26.6 /   -  / 47.1 / 84.5
//                         256:  72.6 /   -  / 38.1 / 29.0 / 25.1 / 35.4 / 96.9
//                         512:    -  /   -  / 68.9 / 56.6 / 46.7 / 41.3 / 86.6
//                        2048:    -  /   -  /   -  /  223 /   -  /  152 /  118
//                        8192:    -  /   -  /   -  /  903 /   -  /  599 /  437 (a library int8 product 439)
//         28,672 of 8192,  20:  62.1 / 39.3 / 36.5 / 39.6 / 59.0 / 51.0 / 83.5
//         151,936 of 2048, 20:  86.0 / 53.2 / 52.2 / 57.1 / 78.9 / 55.8 / 78.4
//                          64:   145 / 91.2 / 90.5 / 80.3 / 86.5 / 72.4 / 94.4   (fp32)
//                         128:   261 /  150 /  135 /  107 / 90.4 / 83.6 / 92.5
//                         200:   404 /  234 /  198 /  177 /  144 /  119 /  105
int launch_product(const moe_i8_linear *L, const int8_t *codes, int64_t pitch, const float *scales, int columns, void *y,
                   int y_type, int64_t y_stride, hipStream_t s) {
    moe::I8Args a{};
    a.blocks = L->mem;
    a.sw = L->scales;
    a.x = codes;
    a.sx = scales;
    a.pitch = pitch;
    a.x_rows = columns;
    a.experts = 1;
    a.y = y;
    a.y_stride = y_stride;
    a.M = L->output;
    a.rows = moe::i8_rows(L->output);
    a.N = columns;
    a.K = L->input;
    a.chunks = moe::i8_chunks(L->input);
    const auto tiles = [&](long m, long n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    if (a.N <= moe::kFewRows) return moe::launch_few<moe::kCodes>(few_args(L, codes, pitch, scales, columns, y, y_type, y_stride, nullptr), s);
    const long t256 = tiles(256, 256);
    if (a.N > 128 && t256 * 5 >= 3 * 256 * ((t256 + 255) / 256)) return launch_gemm<2, 4, 8, 4, 4, 1>(a, y_type, s);
    const long t128 = tiles(64, 128);
    if (a.N > 32 && t128 > 256) return launch_gemm<4, 2, 2, 4, 4, 1>(a, y_type, s);
    if (a.N > 64 && t128 >= 150) return launch_gemm<2, 4, 2, 2, 4, 2>(a, y_type, s);
    if (tiles(64, 16) <= 256) return launch_gemm<4, 1, 1, 1, 4, 4>(a, y_type, s);
    if (tiles(64, 32) <= 256) return launch_gemm<2, 2, 2, 1, 4, 4>(a, y_type, s);
    if (a.N <= 32) return launch_gemm<2, 2, 2, 1, 4, 2>(a, y_type, s);
    return launch_gemm<2, 4, 2, 1, 4, 2>(a, y_type, s);
}

}  // namespace

extern "C" {

int moe_quantize_i8(const void *x, int x_type, int64_t x_stride, int width, int columns, void *codes, float *scales,
                    int *error, void *stream) {
    if (width < 1 || width > 16384 || columns < 1 || columns > 65536 || !valid_rows(x, x_type, x_stride, width) || !codes ||
        !aligned(scales, 4) || !aligned(error, 4))
        return kInvalid;
    const moe::I8Rows r{x, x_stride, width, static_cast<size_t>(columns), static_cast<int8_t *>(codes), width, scales, error};
    return moe::launch_quantize_i8(r, x_type, static_cast<hipStream_t>(stream));
}

int moe_i8_linear_create(int input, int output, int max_columns, const void *codes, const float *scales,
                         int weights_on_device, int device, moe_i8_linear **out) {
    if (!out) return kInvalid;
    *out = nullptr;
    if (input < 32 || input > 16384 || input % 32 || output < 1 || output > 262144 || max_columns < 0 || max_columns > 65536 ||
        !codes || !aligned(scales, 4) || device < 0)
        return kInvalid;
    moe::DeviceScope scope(device);
    if (!scope.ok()) return hipErrorInvalidDevice;
    auto *L = new (std::nothrow) moe_i8_linear;
    if (!L) return hipErrorOutOfMemory;
    L->input = input;
    L->output = output;
    L->max_columns = max_columns;
    L->device = device;
    // Rows an odd number of 64 bytes apart, so that those of one load do not share
    // a memory channel.
    L->pitch = (moe::i8_chunks(input) | 1) * moe::kI8Chunk;
    const size_t code_bytes = static_cast<size_t>(output) * input;
    const size_t scale_at = static_cast<size_t>(moe::i8_rows(output)) * moe::i8_chunks(input) * moe::kI8Chunk;
    const size_t scale_bytes = static_cast<size_t>(output) * 4;
    void *staging = nullptr;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, scale_at + moe::i8_rows(output) * sizeof(float));
    if (r == hipSuccess && max_columns > 0) r = hipMalloc(&L->ws, static_cast<size_t>(max_columns) * (L->pitch + 4));
    const void *device_codes = codes;
    if (r == hipSuccess && !weights_on_device) {
        r = hipMalloc(&staging, code_bytes);
        if (r == hipSuccess) r = hipMemcpy(staging, codes, code_bytes, hipMemcpyHostToDevice);
        device_codes = staging;
    }
    if (r == hipSuccess)
        r = moe::launch_i8_repack(static_cast<const int8_t *>(device_codes), L->mem, 1, output, input, moe::kI8Whole, nullptr);
    if (r == hipSuccess)
        r = hipMemcpy(L->mem + scale_at, scales, scale_bytes, weights_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (staging) (void)hipFree(staging);
    if (r != hipSuccess) { release(L); return r; }
    L->scales = reinterpret_cast<const float *>(L->mem + scale_at);
    *out = L;
    return 0;
}

int moe_i8_linear_destroy(moe_i8_linear *L) {
    if (!L) return kInvalid;
    moe::DeviceScope scope(L->device);
    release(L);
    return 0;
}

int moe_i8_linear_bytes(const moe_i8_linear *L, size_t *weight_bytes) {
    if (!L || !weight_bytes) return kInvalid;
    *weight_bytes = static_cast<size_t>(L->output) * (static_cast<size_t>(L->input) + 4);
    return 0;
}

int moe_i8_linear_forward(moe_i8_linear *L, const void *x_codes, const float *x_scales, int columns, void *y, int y_type,
                          int64_t y_stride, void *stream) {
    if (!L || !aligned(x_codes, 16) || !aligned(x_scales, 4) || columns < 1 || columns > 65536 ||
        !valid_rows(y, y_type, y_stride, L->output))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    return launch_product(L, static_cast<const int8_t *>(x_codes), L->input, x_scales, columns, y, y_type, y_stride,
                          static_cast<hipStream_t>(stream));
}

int moe_i8_linear_apply(moe_i8_linear *L, const void *x, int x_type, int64_t x_stride, int columns, void *y, int y_type,
                        int64_t y_stride, int *error, void *stream) {
    if (!L || columns < 1 || columns > L->max_columns || !valid_rows(x, x_type, x_stride, L->input) ||
        !valid_rows(y, y_type, y_stride, L->output) || !aligned(error, 4))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    const auto s = static_cast<hipStream_t>(stream);
    const auto extent = [&](int64_t stride, int width, int type) {
        return (static_cast<size_t>(columns - 1) * stride + width) * moe::elem_bytes(type);
    };
    const char *xb = static_cast<const char *>(x), *yb = static_cast<const char *>(y);
    const bool apart = xb + extent(x_stride, L->input, x_type) <= yb || yb + extent(y_stride, L->output, y_type) <= xb;
    // Every workgroup (16 outputs) quantises all of the rows: in the product's kernel where
    // each thread has few vectors of them and all workgroups are on the chip at once (4 a
    // CU), up to 16,384 outputs; with more than four rows, to 2^26 products.  us, so / in two
    // launches, bf16:
    //   outputs                2,048      8,192      16,384     32,768     65,536     151,936
    //   input 512, 1 row     4.0 / 6.6  4.4 / 6.7  6.0 / 6.5  9.9 / 7.1  16.9 / 9.7  35.3 / 17.2
    //              4         4.0 / 6.5  4.4 / 6.5  6.1 / 6.4  10.3 / 6.9 17.6 / 9.6  37.5 / 17.5
    //             16         4.2 / 6.4  5.0 / 6.5  7.3 / 6.5  13.0 / 7.3 22.4 / 10.6 49.6 / 20.1
    //   2,048,     1         4.1 / 6.6  5.7 / 6.8  8.7 / 9.3  14.4 / 15.1 24.0 / 25.0 49.9 / 49.2
    //              4         4.4 / 6.4  6.3 / 6.9  9.3 / 9.4  16.5 / 15.3 27.9 / 25.4 59.5 / 50.9
    //              8         4.9 / 6.5  7.5 / 7.1  11.5 / 9.6 20.1 / 15.7 34.7 / 26.2 75.9 / 53.7
    //   8,192,     2         8.2 / 12.3 14.7 / 18.2 27.6 / 26.2 45.6 / 46.7 85.9 / 86.5 191 / 193
    const bool in_one = columns * L->input <= kFewElements && L->output <= kFewOutputs &&
                        (columns <= 4 || columns * L->input * L->output <= 1 << 26);
    if (columns <= moe::kFewRows && apart && in_one) {
        const moe::I8FewArgs f = few_args(L, x, x_stride, nullptr, columns, y, y_type, y_stride, error);
        if (x_type == MOE_F32) return moe::launch_few<moe::kF32>(f, s);
        if (x_type == MOE_BF16) return moe::launch_few<moe::kBF16>(f, s);
        return moe::launch_few<moe::kF16>(f, s);
    }
    auto *scales = reinterpret_cast<float *>(L->ws + static_cast<size_t>(columns) * L->pitch);
    const moe::I8Rows rows{x, x_stride, L->input, static_cast<size_t>(columns), L->ws, L->pitch, scales, error};
    const hipError_t r = moe::launch_quantize_i8(rows, x_type, s);
    if (r != hipSuccess) return r;
    return launch_product(L, L->ws, L->pitch, scales, columns, y, y_type, y_stride, s);
}

}  // extern "C"
