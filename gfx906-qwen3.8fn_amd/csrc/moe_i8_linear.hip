// Matrices of int8 codes with one fp32 scale per output channel
// (moe_i8_linear_*) and the quantiser of their activations.
#include "moe_ffn.h"
#include "moe_i8.hpp"

#include <algorithm>
#include <new>

namespace moe {
namespace {

// --------------------------------------------------------------- layout ---
// One thread per 16-byte piece of the tiles of `rows` rows (of matrices of `period`
// rows each, a multiple of 16 where pairs is set).
__global__ __launch_bounds__(256) void k_i8_repack(const int8_t *__restrict__ codes, uint4 *__restrict__ tiles, int rows,
                                                   int cols, int chunks, size_t pieces, int pairs, int shift) {
    const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int lane = static_cast<int>(i & 63), row_tiles = (rows + 15) / 16;
    const size_t tile = i >> 6, chunk = tile % chunks, at = tile / chunks;   // at: row tile over all matrices
    const size_t matrix = at / row_tiles;
    const int row = static_cast<int>(at % row_tiles) * 16 + (lane & 15), col = static_cast<int>(chunk) * kI8Chunk + (lane >> 4) * 16;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows && col < cols) __builtin_memcpy(&v, codes + (matrix * rows + row) * cols + col, 16);
    tiles[((pairs ? at * 2 + shift : at) * chunks + chunk) * 64 + lane] = v;
}

// ------------------------------------------------------------- quantiser ---
// A row's elements stay in the registers of its L lanes (a wave, or the whole
// workgroup), V times eight of them a lane, between the maximum and the codes.
template<int T, int L, int V>
__global__ __launch_bounds__(256) void k_quantize_i8(const void *__restrict__ x, int64_t stride, int width, size_t rows,
                                                     int8_t *__restrict__ codes, int64_t pitch, float *__restrict__ scales,
                                                     int *error) {
    const size_t n = static_cast<size_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
    const int l = threadIdx.x % L;
    const bool there = n < rows;   // whole waves
    Raw8 raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = (i * L + l) * 8;
        raw[i] = load8_any<T>(x, (there ? n : 0) * static_cast<size_t>(stride) + k, there ? width - k : 0);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float v[8];
        unpack8<T>(raw[i], v);
#pragma unroll
        for (int q = 0; q < 8; ++q) m = max(m, magnitude(v[q]));
    }
    const auto larger = [](uint32_t a, int b) { return max(a, static_cast<uint32_t>(b)); };
    m = larger(m, lane_xor<1>(static_cast<int>(m)));
    m = larger(m, lane_xor<2>(static_cast<int>(m)));
    m = larger(m, lane_xor<4>(static_cast<int>(m)));
    m = larger(m, lane_xor<8>(static_cast<int>(m)));
    m = larger(m, lane_xor<16>(static_cast<int>(m)));
    m = larger(m, lane_xor<32>(static_cast<int>(m)));
    if constexpr (L > 64) {
        __shared__ uint32_t most[L / 64];
        if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < L / 64; ++w) m = max(m, most[w]);
    }
    if (!there) return;
    const GroupScale s = row_scale(m);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = (i * L + l) * 8;
        if (k >= width) break;
        float v[8];
        unpack8<T>(raw[i], v);
        const uint2 c = quantize8_i8(v, s);
        int8_t *out = codes + n * static_cast<size_t>(pitch) + k;
        if (k + 8 <= width) {
            __builtin_memcpy(out, &c, 8);
        } else {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (k + q < width) out[q] = static_cast<int8_t>((q < 4 ? c.x : c.y) >> (8 * (q & 3)));
        }
    }
    if (l == 0) {
        scales[n] = s.s;
        if (s.bad) atomicOr(error, 1);
    }
}

template<int T>
void launch_quantize(const void *x, int64_t stride, int width, size_t rows, int8_t *codes, int64_t pitch, float *scales,
                     int *error, hipStream_t s) {
    const auto launch = [&](auto kernel, int lanes) {
        const size_t per = 256 / lanes;
        kernel<<<dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0, s>>>(x, stride, width, rows, codes, pitch,
                                                                                         scales, error);
    };
    if (width <= 512) launch(k_quantize_i8<T, 64, 1>, 64);
    else if (width <= 1024) launch(k_quantize_i8<T, 64, 2>, 64);
    else if (width <= 2048) launch(k_quantize_i8<T, 256, 1>, 256);
    else if (width <= 4096) launch(k_quantize_i8<T, 256, 2>, 256);
    else if (width <= 8192) launch(k_quantize_i8<T, 256, 4>, 256);
    else launch(k_quantize_i8<T, 256, 8>, 256);
}

}  // namespace

hipError_t launch_i8_repack(const int8_t *codes, uint8_t *tiles, size_t matrices, int rows, int cols, bool pairs, int shift,
                            hipStream_t s) {
    const int chunks = i8_chunks(cols), row_tiles = (rows + 15) / 16;
    // A grid holds fewer than 2^32 threads: at most 2^30 pieces a launch.
    const size_t each = static_cast<size_t>(row_tiles) * chunks * 64, at_once = std::max<size_t>(1, (size_t{1} << 30) / each);
    for (size_t first = 0; first < matrices; first += at_once) {
        const size_t n = std::min(at_once, matrices - first), pieces = n * each;
        k_i8_repack<<<dim3(static_cast<unsigned>((pieces + 255) / 256)), dim3(256), 0, s>>>(
            codes + first * rows * cols, reinterpret_cast<uint4 *>(tiles + first * each * 16 * (pairs ? 2 : 1)), rows, cols,
            chunks, pieces, pairs ? 1 : 0, shift);
    }
    return hipGetLastError();
}

hipError_t launch_quantize_i8(const void *x, int type, int64_t stride, int width, size_t rows, int8_t *codes, int64_t pitch,
                              float *scales, int *error, hipStream_t s) {
    if (type == kF32) launch_quantize<kF32>(x, stride, width, rows, codes, pitch, scales, error, s);
    else if (type == kBF16) launch_quantize<kBF16>(x, stride, width, rows, codes, pitch, scales, error, s);
    else launch_quantize<kF16>(x, stride, width, rows, codes, pitch, scales, error, s);
    return hipGetLastError();
}

namespace {

// Tile t of an output of tm x tn tiles: workgroup i runs on XCD i % 8, whose L2 the
// others do not see, so each XCD takes a run of tiles of its own, in columns of
// eight tiles of the matrix.
struct TileAt {
    int m, n;
};
__device__ __forceinline__ TileAt tile_of(int t, int tm, int tn) {
    constexpr int P = 8;
    const int panel = t / (P * tn), r = t - panel * P * tn, p = min(P, tm - panel * P);
    return TileAt{panel * P + r % p, r / p};
}

template<int WR, int WC, int TM, int TN, int S, int KS, int Y>
__global__ __launch_bounds__(64 * WR * WC) void k_i8_gemm(I8Args a) {
    using Tile = I8Tile<WR, WC, TM, TN, S, KS>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::Lds];
    const int tn = (a.N + Tile::BN - 1) / Tile::BN, total = a.tiles_m * tn, each = (total + 7) / 8;
    const int t = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if (static_cast<int>(blockIdx.x >> 3) >= each || t >= total) return;
    const TileAt at = tile_of(t, a.tiles_m, tn);
    const int m0 = at.m * Tile::BM, n0 = at.n * Tile::BN, cols = min(a.N - n0, Tile::BN);
    Tile g(lds);
    int flags = 0;
    g.start(a, 0, m0, n0, cols, flags);
    i32x4 acc[TM][TN];
    g.product(lds, acc);
    g.template store_rows<Y>(a, 0, m0, n0, cols, acc, lds);
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_i8_linear {
    int input = 0, output = 0, max_columns = 0, device = 0;
    uint8_t *mem = nullptr;   // tiles, scales
    const float *scales = nullptr;
    int8_t *ws = nullptr;     // rows of `pitch` codes, then their scales
    int64_t pitch = 0;
};

namespace {

constexpr int kInvalid = hipErrorInvalidValue;

bool aligned(const void *p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }
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

template<int WR, int WC, int TM, int TN, int S, int KS>
int launch_gemm(moe::I8Args a, int y_type, hipStream_t s) {
    using Tile = moe::I8Tile<WR, WC, TM, TN, S, KS>;
    a.tiles_m = (a.M + Tile::BM - 1) / Tile::BM;
    const size_t total = static_cast<size_t>(a.tiles_m) * ((a.N + Tile::BN - 1) / Tile::BN);
    const dim3 grid(static_cast<unsigned>((total + 7) / 8 * 8)), block(64 * Tile::W);
    if (y_type == MOE_F32) moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kF32><<<grid, block, 0, s>>>(a);
    else if (y_type == MOE_BF16) moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kBF16><<<grid, block, 0, s>>>(a);
    else moe::k_i8_gemm<WR, WC, TM, TN, S, KS, moe::kF16><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

int launch_product(const moe_i8_linear *L, const int8_t *codes, int64_t pitch, const float *scales, int columns, void *y,
                   int y_type, int64_t y_stride, hipStream_t s) {
    moe::I8Args a{};
    a.tiles = L->mem;
    a.sw = L->scales;
    a.x = codes;
    a.sx = scales;
    a.pitch = pitch;
    a.x_rows = columns;
    a.experts = 1;
    a.y = y;
    a.y_stride = y_stride;
    a.M = L->output;
    a.N = columns;
    a.K = L->input;
    a.chunks = moe::i8_chunks(L->input);
    const auto tiles = [&](long m, long n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    if (a.N <= 16) return launch_gemm<4, 1, 1, 1, 3, 4>(a, y_type, s);
    if (tiles(128, 128) < 400) return launch_gemm<2, 2, 2, 2, 3, 2>(a, y_type, s);
    if (tiles(256, 256) < 256) return launch_gemm<2, 2, 4, 4, 4, 1>(a, y_type, s);
    return launch_gemm<2, 2, 8, 8, 4, 1>(a, y_type, s);
}

}  // namespace

extern "C" {

int moe_quantize_i8(const void *x, int x_type, int64_t x_stride, int width, int columns, void *codes, float *scales,
                    int *error, void *stream) {
    if (width < 1 || width > 16384 || columns < 1 || columns > 65536 || !valid_rows(x, x_type, x_stride, width) || !codes ||
        !aligned(scales, 4) || !aligned(error, 4))
        return kInvalid;
    return moe::launch_quantize_i8(x, x_type, x_stride, width, columns, static_cast<int8_t *>(codes), width, scales, error,
                                   static_cast<hipStream_t>(stream));
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
    const size_t tiles = static_cast<size_t>((output + 15) / 16) * moe::i8_chunks(input) * moe::kI8TileBytes;
    const size_t scale_at = round_up(tiles, 256), scale_bytes = static_cast<size_t>(output) * 4;
    void *staging = nullptr;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, scale_at + scale_bytes);
    if (r == hipSuccess && max_columns > 0) r = hipMalloc(&L->ws, static_cast<size_t>(max_columns) * (L->pitch + 4));
    const void *device_codes = codes;
    if (r == hipSuccess && !weights_on_device) {
        r = hipMalloc(&staging, code_bytes);
        if (r == hipSuccess) r = hipMemcpy(staging, codes, code_bytes, hipMemcpyHostToDevice);
        device_codes = staging;
    }
    if (r == hipSuccess)
        r = moe::launch_i8_repack(static_cast<const int8_t *>(device_codes), L->mem, 1, output, input, false, 0, nullptr);
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
    auto *scales = reinterpret_cast<float *>(L->ws + static_cast<size_t>(columns) * L->pitch);
    const hipError_t r = moe::launch_quantize_i8(x, x_type, x_stride, L->input, columns, L->ws, L->pitch, scales, error, s);
    if (r != hipSuccess) return r;
    return launch_product(L, L->ws, L->pitch, scales, columns, y, y_type, y_stride, s);
}

}  // extern "C"
