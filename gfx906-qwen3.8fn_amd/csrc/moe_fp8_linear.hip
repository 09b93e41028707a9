// Matrices of e4m3 values with one fp32 scale per block of 128 x 128
// (moe_fp8_linear_*) and the quantiser of their activations:
//   y[n][m] = sum_b sx[n][b] sw[m / 128][b] sum_{k in block b} cx[n][k] cw[m][k]
// The inner sum is one MFMA tile step; its result is multiplied by both
// scales into an fp32 accumulator, and y is rounded once.
#include "moe_ffn.h"
#include "moe_fp8.hpp"

#include <algorithm>
#include <new>
#include <type_traits>

namespace moe {
namespace {

// --------------------------------------------------------------- layout ---
// One thread per 16-byte chunk of the tiles.
__global__ __launch_bounds__(256) void k_fp8_repack(const uint8_t *__restrict__ codes, uint4 *__restrict__ tiles,
                                                    size_t rows, int cols, int nb, size_t chunks) {
    const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= chunks) return;
    const int lane = static_cast<int>(i & 63), half = static_cast<int>(i >> 6) & 1;
    const size_t tile = i >> 7;
    const size_t row = tile / nb * kFp8TileRows + (lane & 15);
    const int col = static_cast<int>(tile % nb) * kFp8Block + (lane >> 4) * 32 + half * 16;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows && col < cols) __builtin_memcpy(&v, codes + row * cols + col, 16);
    tiles[i] = v;
}

// ------------------------------------------------------------- quantiser ---
// 16 lanes per group of 128, 8 elements each; bound by memory (16,384 rows of 8,192
// bf16 elements 73 us, 5.5 TB/s, at any alignment of the rows: one odd element
// away 2,048 take 22.1 us against 21.3, element by element they took 54).
// Tiles: a workgroup writes one tile (16 rows, one block) of the products'
// operand layout, and scales [block][row]; otherwise the canonical rows.
template<int T, bool Tiles>
__global__ __launch_bounds__(256) void k_quantize_e4m3(const void *__restrict__ x, int64_t stride, int width, int nb,
                                                       int columns, uint8_t *__restrict__ codes,
                                                       float *__restrict__ scales, int64_t scale_stride, int *error) {
    size_t n;
    int b;
    const int part = threadIdx.x & 15;
    if constexpr (Tiles) {
        n = static_cast<size_t>(blockIdx.x / nb) * 16 + (threadIdx.x >> 4);
        b = blockIdx.x % nb;
    } else {
        const size_t g = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;
        n = g / nb;
        b = static_cast<int>(g % nb);
    }
    if (n >= static_cast<size_t>(columns)) return;   // whole groups of 16 lanes
    const int k = b * kFp8Block + part * 8;
    const size_t at = n * static_cast<size_t>(stride) + k;
    float v[8];
    unpack8<T>(load8_any<T>(x, at, width - k), v);
    const GroupScale s = group_scale(max16(v));
    const uint2 c = quantize8(v, s);
    if constexpr (Tiles) {
        // Elements 8 part .. + 7: half of a chunk of lane 16 (part / 4) + n % 16.
        uint8_t *tile = codes + (n / 16 * nb + b) * kFp8TileBytes;
        *reinterpret_cast<uint2 *>(tile + tile_offset(part, static_cast<int>(n & 15))) = c;
        if (part == 0) scales[b * scale_stride + n] = s.s;
    } else {
        uint8_t *out = codes + n * width + k;
        if (k + 8 <= width) {
            __builtin_memcpy(out, &c, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (k + i < width) out[i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
        }
        if (part == 0) scales[n * nb + b] = s.s;
    }
    if (part == 0 && s.bad) atomicOr(error, 1);
}

}  // namespace

hipError_t launch_fp8_repack(const uint8_t *codes, uint8_t *tiles, size_t rows, int cols, hipStream_t s) {
    const int nb = (cols + kFp8Block - 1) / kFp8Block;
    // A grid holds fewer than 2^32 threads: at most 2^30 chunks a launch.
    const size_t row_chunks = static_cast<size_t>(nb) * kFp8TileBytes / 16;   // of 16 rows
    const size_t rows_at_once = (size_t{1} << 30) / row_chunks * kFp8TileRows;
    for (size_t first = 0; first < rows; first += rows_at_once) {
        const size_t n = std::min(rows_at_once, rows - first);
        const size_t chunks = (n + kFp8TileRows - 1) / kFp8TileRows * row_chunks;
        k_fp8_repack<<<dim3(static_cast<unsigned>((chunks + 255) / 256)), dim3(256), 0, s>>>(
            codes + first * cols, reinterpret_cast<uint4 *>(tiles + first / kFp8TileRows * nb * kFp8TileBytes), n, cols, nb,
            chunks);
    }
    return hipGetLastError();
}

namespace {

template<bool Tiles>
hipError_t launch_quantize(const void *x, int type, int64_t stride, int width, int columns, uint8_t *codes,
                           float *scales, int64_t scale_stride, int *error, hipStream_t s) {
    const int nb = (width + kFp8Block - 1) / kFp8Block;
    const size_t groups = Tiles ? static_cast<size_t>((columns + 15) / 16) * nb : (static_cast<size_t>(columns) * nb + 15) / 16;
    const dim3 grid(static_cast<unsigned>(groups)), block(256);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, block, 0, s>>>(x, stride, width, nb, columns, codes, scales, scale_stride, error);
    };
    if (type == kF32) launch(k_quantize_e4m3<kF32, Tiles>);
    else if (type == kBF16) launch(k_quantize_e4m3<kBF16, Tiles>);
    else launch(k_quantize_e4m3<kF16, Tiles>);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_e4m3(const void *x, int type, int64_t stride, int width, int columns, uint8_t *codes,
                                float *scales, int *error, hipStream_t s) {
    return launch_quantize<false>(x, type, stride, width, columns, codes, scales, 0, error, s);
}

namespace {

struct Fp8LinearArgs {
    const uint8_t *tiles;    // [ceil(M/16)][nb] tiles
    const float *wscale;     // [ceil(M/128)][nb]
    const void *x;           // rows of a type (few columns), or unused
    int64_t x_stride;
    const uint8_t *codes;    // e4m3 columns: rows [N][K], or tiles [ceil(N/16)][nb]
    const float *xscale;     // scale of column n, block b at n scale_n + b scale_b
    int scale_n, scale_b;
    void *y;
    int64_t y_stride;
    int y_type;
    int M, N, K, nb;
    int *error;
};

// Four results of one token, rows m .. m + 3.
template<int Y>
__device__ __forceinline__ void store_rows(const Fp8LinearArgs &a, int n, int m, const float (&v)[4]) {
    const size_t at = static_cast<size_t>(n) * a.y_stride + m;
    if (m + 3 < a.M) {
        store4<Y>(a.y, at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (m + i < a.M) store1<Y>(a.y, at + i, v[i]);
}
__device__ __forceinline__ void store_rows(const Fp8LinearArgs &a, int n, int m, const float (&v)[4]) {
    if (a.y_type == kF32) store_rows<kF32>(a, n, m, v);
    else if (a.y_type == kBF16) store_rows<kBF16>(a, n, m, v);
    else store_rows<kF16>(a, n, m, v);
}

// All of the columns (at most 16) quantised by the whole workgroup into LDS:
// codes [block][32-element part][column][32 B], scales [block][column], 16
// threads a block.  Elements past a row's end count as zero.
template<int T>
__device__ __forceinline__ void quantize_to_lds(const Fp8LinearArgs &a, uint8_t *codes, float *scales, int &flags) {
    const int part = threadIdx.x & 15;
    for (int i = threadIdx.x >> 4; i < a.N * a.nb; i += blockDim.x >> 4) {
        const int n = i / a.nb, b = i % a.nb, k = b * kFp8Block + part * 8;
        const size_t at = static_cast<size_t>(n) * a.x_stride + k;
        float v[8];
        unpack8<T>(load8_any<T>(a.x, at, a.K - k), v);
        const GroupScale s = group_scale(max16(v));
        *reinterpret_cast<uint2 *>(codes + ((b * 4 + (part >> 2)) * a.N + n) * 32 + (part & 3) * 8) = quantize8(v, s);
        if (part == 0) scales[b * a.N + n] = s.s;
        if (s.bad) flags |= 1;
    }
}

// Few columns: a workgroup takes 16 RT rows and 16 NT columns, its waves share
// out the blocks of the row (wave w: blocks w, w + W, ..) and add up through
// LDS in wave order.  The matrix streams from memory straight into registers,
// each tile once per column tile group; with more than one column tile the
// columns' codes are most of what is read (from L2), which RT = 2 halves.
// IN: the columns' type, quantised here (one column tile), or kCodes (rows), kTiles.
template<int IN, int NT, int RT>
__global__ __launch_bounds__(512) void k_fp8_stream(Fp8LinearArgs a) {
    constexpr bool Quantize = IN != kCodes && IN != kTiles;
    static_assert(!Quantize || NT == 1);
    __shared__ f32x4 red[8][RT * NT][64];
    extern __shared__ __attribute__((aligned(16))) uint8_t columns[];   // Quantize: codes, then scales
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int W = blockDim.x >> 6, n0 = blockIdx.y * 16 * NT, row_tiles = (a.M + 15) / 16;
    const uint8_t *row[RT];
    const float *wscale[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int mt = min(static_cast<int>(blockIdx.x) * RT + r, row_tiles - 1);   // past the end: the last one again
        row[r] = a.tiles + static_cast<size_t>(mt) * a.nb * kFp8TileBytes;
        wscale[r] = a.wscale + static_cast<size_t>(mt * kFp8TileRows / kFp8Block) * a.nb;
    }
    const int kl = (lane >> 4) * 32;
    int token[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) token[t] = min(n0 + 16 * t + (lane & 15), a.N - 1);
    f32x4 acc[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int flags = 0;
    constexpr int U = NT == 1 ? 4 : 2;   // blocks whose loads are in flight together
    const float *scales = reinterpret_cast<const float *>(columns + static_cast<size_t>(a.N) * a.nb * kFp8Block);
    Frag w[U][RT];
    const auto load = [&](int b0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Past the last block: the first one of the round again, not used below.
            const int b = b0 + u * W < a.nb ? b0 + u * W : b0;
#pragma unroll
            for (int r = 0; r < RT; ++r) w[u][r] = load_tile(row[r] + static_cast<size_t>(b) * kFp8TileBytes, lane);
        }
    };
    if constexpr (Quantize) {
        load(wave);
        quantize_to_lds<IN>(a, columns, const_cast<float *>(scales), flags);
        __syncthreads();
    }
    for (int b0 = wave; b0 < a.nb; b0 += W * U) {
        if (!Quantize || b0 != wave) load(b0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * W;
            if (b >= a.nb) break;
            FragF16 wf[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) wf[r] = to_f16(w[u][r]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                Frag x;
                float sx;
                if constexpr (IN == kTiles) {
                    const int tile = min(n0 / 16 + t, (a.N - 1) / 16);
                    x = load_tile(a.codes + (static_cast<size_t>(tile) * a.nb + b) * kFp8TileBytes, lane);
                } else if constexpr (IN == kCodes) {
                    const int k = b * kFp8Block + kl;
                    x = Frag{};
                    if (k < a.K) {
                        const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + static_cast<size_t>(token[t]) * a.K + k);
                        x = Frag{p[0], p[1]};
                    }
                } else {
                    const int n = min(lane & 15, a.N - 1);
                    const uint4 *p = reinterpret_cast<const uint4 *>(columns + ((b * 4 + (lane >> 4)) * a.N + n) * 32);
                    x = Frag{p[0], p[1]};
                    sx = scales[b * a.N + n];
                }
                if constexpr (!Quantize)
                    sx = a.xscale[static_cast<size_t>(token[t]) * a.scale_n + static_cast<size_t>(b) * a.scale_b];
                const FragF16 xf = to_f16(x);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const f32x4 p = block_dot(wf[r], xf);
                    const float s = sx * wscale[r][b];
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][t][i] = fmaf(p[i], s, acc[r][t][i]);
                }
            }
        }
    }
    if constexpr (Quantize) {
        if (blockIdx.x == 0 && flags) atomicOr(a.error, flags);   // every workgroup quantises the same columns
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) red[wave][r * NT + t][lane] = acc[r][t];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * RT * NT; i += blockDim.x) {
        const int q = i >> 6, r = q / NT, t = q % NT, l = i & 63;
        f32x4 s = red[0][q][l];
        for (int j = 1; j < W; ++j) {
            const f32x4 v = red[j][q][l];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = s[e] + v[e];
        }
        const int n = n0 + 16 * t + (l & 15);
        const float v[4] = {s[0], s[1], s[2], s[3]};
        if (n < a.N) store_rows(a, n, (static_cast<int>(blockIdx.x) * RT + r) * kFp8TileRows + (l >> 4) * 4, v);
    }
}

// Few tiles: W waves share the blocks of 16 TM rows x 16 TN columns (wave w:
// blocks w, w + W, ..), each with its operands straight from memory into
// registers, the next block's on their way during a block, and no barrier
// before the sums meet in LDS in wave order.  Nothing but the sums is shared, so
// that every operand crosses the L1 once for each tile: this pays while a CU's
// tiles are few (2080 x 1000 at 333 canonical rows, bf16 results: 7.8 us as 64 x 64
// tiles through LDS, 5.9 so) and, on tiles of columns, for fp32 results, whose
// conversions leave the L1 the time (the table at launch_product).  Canonical
// rows, a power of two apart and with a scale load each, do not come fast enough
// for more: 2048 x 2048 at 1,032 columns, fp32, in 32 x 48 tiles 34.5 us against
// 20.9.
// Y: type of y; Sums32: fp32 sums within a block (block_dot), as fp32 results always have.
template<int TM, int TN, int W, bool Tiles, int Y, bool Sums32>
__global__ __launch_bounds__(64 * W) void k_fp8_split(Fp8LinearArgs a, int tiles_m) {
    static_assert(kFp8Block % (16 * TM) == 0, "the rows share one scale block");
    static_assert(Sums32 || Y != kF32);
    using Operand = std::conditional_t<Sums32, FragF16, Frag>;
    __shared__ f32x4 red[W][TM * TN][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int mt = static_cast<int>(blockIdx.x) % tiles_m * TM, nt = static_cast<int>(blockIdx.x) / tiles_m * TN;
    const int row_tiles = (a.M + 15) / 16, col_tiles = (a.N + 15) / 16, kl = (lane >> 4) * 32;
    // Tiles past the end: the last one again, not stored.
    const uint8_t *row[TM], *col[TN];
    const float *xscale[TN], *wscale = a.wscale + static_cast<size_t>(mt * kFp8TileRows / kFp8Block) * a.nb;
#pragma unroll
    for (int i = 0; i < TM; ++i)
        row[i] = a.tiles + static_cast<size_t>(min(mt + i, row_tiles - 1)) * a.nb * kFp8TileBytes;
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        const int n = min((nt + t) * 16 + (lane & 15), a.N - 1);
        if constexpr (Tiles) col[t] = a.codes + static_cast<size_t>(min(nt + t, col_tiles - 1)) * a.nb * kFp8TileBytes;
        else col[t] = a.codes + static_cast<size_t>(n) * a.K + kl;
        xscale[t] = a.xscale + static_cast<size_t>(n) * a.scale_n;
    }
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Frag w[TM], x[TN];   // of the next block
    float sx[TN];
    const auto load_row = [&](int i, int b) { w[i] = load_tile(row[i] + static_cast<size_t>(b) * kFp8TileBytes, lane); };
    const auto load_column = [&](int t, int b) {
        if constexpr (Tiles) {
            x[t] = load_tile(col[t] + static_cast<size_t>(b) * kFp8TileBytes, lane);
        } else {
            x[t] = Frag{};
            if (b * kFp8Block + kl < a.K) {
                const uint4 *p = reinterpret_cast<const uint4 *>(col[t] + b * kFp8Block);
                x[t] = Frag{p[0], p[1]};
            }
        }
        sx[t] = xscale[t][static_cast<size_t>(b) * a.scale_b];
    };
    if (wave < a.nb) {
#pragma unroll
        for (int t = 0; t < TN; ++t) load_column(t, wave);
#pragma unroll
        for (int i = 0; i < TM; ++i) load_row(i, wave);
    }
    for (int b = wave; b < a.nb; b += W) {
        const int next = b + W < a.nb ? b + W : b;   // past the last block: it again, not used
        const float sw = wscale[b];
        Operand xo[TN];
        float s[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            xo[t] = operand<Operand>(x[t]);
            s[t] = sx[t] * sw;
            load_column(t, next);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const Operand wo = operand<Operand>(w[i]);
            load_row(i, next);
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const f32x4 p = block_dot(wo, xo[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(p[e], s[t], acc[i][t][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) red[wave][i * TN + t][lane] = acc[i][t];
    __syncthreads();
    for (int q = wave; q < TM * TN; q += W) {
        f32x4 v = red[0][q][lane];
#pragma unroll
        for (int j = 1; j < W; ++j) v += red[j][q][lane];
        const int n = (nt + q % TN) * 16 + (lane & 15);
        const float out[4] = {v[0], v[1], v[2], v[3]};
        if (n < a.N) store_rows<Y>(a, n, (mt + q / TN) * kFp8TileRows + (lane >> 4) * 4, out);
    }
}

// ---------------------------------------------------------- many columns ---
// A workgroup of WR x WC waves takes 16 TM WR rows and 16 TN WC columns, and
// steps through the blocks of K with the next steps' operands and column
// scales on the way to a ring of S buffers in LDS.
//
// Tiles: the columns lie in tiles as the rows do, their scales [block][column].
// Otherwise they are canonical rows with scales [column][block], of which four
// blocks' are loaded at once where a row has that many: a block at a time,
// the columns' scales take as many memory requests as their codes (8192 x 8192
// at 16,384 columns 1.09 ms, in fours 1.01).
template<int WR, int WC, int TM, int TN, int S, int G, bool Tiles>
struct GemmTile {
    static constexpr int W = WR * WC, BM = 16 * TM * WR, BN = 16 * TN * WC;
    static constexpr int ABytes = BM * kFp8Block, BBytes = BN * kFp8Block, Buffer = ABytes + BBytes + BN * 4;
    static constexpr int ALoads = BM / 8 / W, BLoads = BN / 8 / W;   // 1 KiB loads of a wave and step
    static constexpr int Loads = ALoads + BLoads + (Tiles ? 1 : 0);  // at least: and one of scales
    static constexpr int Fours = Tiles ? 0 : 2 * BN * 16;            // two sets of four blocks' scales
    static constexpr int Lds = S * Buffer + Fours;
    static_assert(kFp8Block % (16 * TM) == 0, "a wave's rows share one scale block");
    static_assert(BM / 8 % W == 0 && BN / 8 % W == 0 && W % 2 == 0 && BN % 64 == 0 && W % (BN / 64) == 0,
                  "every wave issues the same loads");

    int lane, wave, wr, wc, m0, n0, K, nb;
    __amdgpu_buffer_rsrc_t ar, br, sr;
    uint32_t tile_row, aoff, boff, boff_last, soff, sstep, lds0;
    // In the constant address space: scalar loads, which the waits above do not count.
    const __attribute__((address_space(4))) float *wscale;
    int b0off, b1off, aread, bread, sread;
    bool fours;   // scales in fours

    __device__ __forceinline__ GemmTile(const Fp8LinearArgs &a, int pm, int pn, const void *lds) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
        wr = wave / WC;
        wc = wave % WC;
        m0 = pm * BM;
        n0 = pn * BN;
        K = a.K;
        nb = a.nb;
        // Rows of the matrix and columns past the end are read as zeros.
        const int row_tiles = (a.M + 15) / 16, cols = min(a.N - n0, BN);
        tile_row = static_cast<uint32_t>(a.nb) * kFp8TileBytes;   // bytes of 16 rows
        ar = buffer_rsrc(a.tiles + static_cast<size_t>(m0 / 16) * tile_row,
                         static_cast<uint32_t>(min(row_tiles - m0 / 16, BM / 16)) * tile_row);
        aoff = lane * 16;
        if constexpr (Tiles) {
            br = buffer_rsrc(a.codes + static_cast<size_t>(n0 / 16) * tile_row, static_cast<uint32_t>((cols + 15) / 16) * tile_row);
        } else {
            // 8 rows of 128 bytes a load, each row's eight chunks permuted by
            // its index so that the fragment reads spread over the LDS banks.
            br = buffer_rsrc(a.codes + static_cast<size_t>(n0) * a.K, static_cast<uint32_t>(cols) * a.K);
            const int bt = lane >> 3, bk = ((lane & 7) ^ bt ^ (wave & 1)) * 16;   // row and byte of the lane's chunk
            boff = static_cast<uint32_t>(bt) * a.K + bk;
            boff_last = (a.nb - 1) * kFp8Block + bk < a.K ? boff : kPastEnd;   // past the row's end: zeros
        }
        // Scales of 64 columns a wave; waves beyond the columns load the same again.
        sr = buffer_rsrc(a.xscale + static_cast<size_t>(n0) * a.scale_n,
                         (static_cast<uint32_t>(cols - 1) * a.scale_n + static_cast<uint32_t>(a.nb - 1) * a.scale_b + 1) * 4);
        soff = static_cast<uint32_t>(wave % (BN / 64) * 64 + lane) * a.scale_n * 4;
        fours = !Tiles && a.nb >= 4;
        sstep = static_cast<uint32_t>(a.scale_b) * 4;
        if (wave % (BN / 64) * 64 + lane >= cols) soff = kPastEnd;
        lds0 = lds_offset(lds);
        wscale = (const __attribute__((address_space(4))) float *)(a.wscale + static_cast<size_t>(min(m0 + wr * 16 * TM, a.M - 1) / kFp8Block) * a.nb);
        if constexpr (!Tiles) {
            // Fragment of column l % 16, chunks 2 (l / 16) and + 1, in the permuted order.
            const int tok = lane & 15, swz = (tok & 7) ^ (tok >> 3), frag = (tok >> 3) * 1024 + (tok & 7) * 128;
            b0off = frag + (((lane >> 4) * 2) ^ swz) * 16;
            b1off = frag + (((lane >> 4) * 2 + 1) ^ swz) * 16;
        }
        aread = wr * TM * 2048;
        bread = ABytes + wc * TN * 2048;
        sread = ABytes + BBytes + (wc * TN * 16 + (lane & 15)) * 4;
    }
    static constexpr uint32_t kPastEnd = 0xc0000000u;   // past every resource here, and no sum with it wraps

    // Start block b's loads into buffer `buf`: the rows, then the columns and
    // their scales.  Past the last block nothing is read (zeros are stored).
    __device__ __forceinline__ void stage_rows(int b, int buf) const {
        const uint32_t to = lds0 + buf * Buffer + wave * 1024;
        const uint32_t off = b < nb ? aoff : kPastEnd;
#pragma unroll
        for (int i = 0; i < ALoads; ++i) {
            const int c = i * W + wave;
            load_to_lds(ar, off + ((c >> 1) * tile_row + b * kFp8TileBytes + (c & 1) * 1024), to + i * W * 1024);
        }
    }
    __device__ __forceinline__ void stage_columns(int b, int buf) const {
        const uint32_t to = lds0 + buf * Buffer + ABytes + wave * 1024;
        const uint32_t off = b >= nb ? kPastEnd : Tiles ? aoff : b + 1 < nb ? boff : boff_last;
#pragma unroll
        for (int i = 0; i < BLoads; ++i) {
            const int c = i * W + wave;
            if constexpr (Tiles)
                load_to_lds(br, off + ((c >> 1) * tile_row + b * kFp8TileBytes + (c & 1) * 1024), to + i * W * 1024);
            else
                load_to_lds(br, off + (8 * c * K + b * kFp8Block), to + i * W * 1024);
        }
        const int part = wave % (BN / 64);
        if (!Tiles && fours) {
            // Of the group's blocks b, b + G, .. the first of each four.
            if ((b & 3) < G)
                load_to_lds(sr, b < nb ? soff + first_of_four(b) * 4 : kPastEnd, lds0 + S * Buffer + (b >> 2 & 1) * (BN * 16) + part * 1024);
        } else {
            load_word_to_lds(sr, b < nb ? soff + b * sstep : kPastEnd, lds0 + buf * Buffer + ABytes + BBytes + part * 256);
        }
    }
    // The first of the four blocks whose scales are loaded with block b's: the
    // last four of a row end with it.
    __device__ __forceinline__ int first_of_four(int b) const { return min(b & ~3, nb - 4); }
    // The scale of column l % 16 of column tile t in block b, whose buffer is buf of lds.
    __device__ __forceinline__ float scale(const uint8_t *lds, const uint8_t *buf, int b, int t) const {
        if (!Tiles && fours)
            return *reinterpret_cast<const float *>(lds + S * Buffer + (b >> 2 & 1) * (BN * 16) + (wc * TN * 16 + t * 16 + (lane & 15)) * 16 + (b - first_of_four(b) & 3) * 4);
        return *reinterpret_cast<const float *>(buf + sread + t * 64);
    }
    __device__ __forceinline__ Frag column(const uint8_t *buf, int t) const {
        const uint8_t *p = buf + bread + t * 2048;
        if constexpr (Tiles) return load_tile(p, lane);
        else return Frag{*reinterpret_cast<const uint4 *>(p + b0off), *reinterpret_cast<const uint4 *>(p + b1off)};
    }
    __device__ __forceinline__ Frag row(const uint8_t *buf, int i) const { return load_tile(buf + aread + i * 2048, lane); }
    // 16-bit results by way of LDS (lds: the buffers, which no wave reads or
    // fills any more), so that a wave's stores run along the rows of y: straight
    // from the accumulators they are pieces of four elements of 16 rows each
    // (96 x 2047 at 16,000 columns 41 us, 22 so; 96 x 2048 26 and 21; 8192 x 8192 at
    // 16,384 1,012 and 985).  fp32 pieces are twice as long: through LDS they took
    // the same time within 4 % in rows of aligned length.  Rows of odd length cost
    // them up to half more (96 x 2047 at 16,000 columns 51 us, 2048 36).
    template<int Y>
    __device__ __forceinline__ void store_along_rows(const Fp8LinearArgs &a, const f32x4 (&acc)[TM][TN], uint8_t *lds) const {
        constexpr int Pitch = BM * 2 + 8, Lanes = BM / 4;   // lanes of a row
        static_assert(G == 1 && Y != kF32 && BN * Pitch <= Lds && 64 * W % Lanes == 0);
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const float v[4] = {acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
                store4<Y>(lds + ((wc * TN + t) * 16 + (lane & 15)) * Pitch, (wr * TM + i) * 16 + (lane >> 4) * 4, v);
            }
        __syncthreads();
        const int c = static_cast<int>(threadIdx.x) % Lanes * 4;
#pragma unroll 4
        for (int n = static_cast<int>(threadIdx.x) / Lanes; n < min(a.N - n0, BN); n += 64 * W / Lanes) {
            uint2 w;
            __builtin_memcpy(&w, lds + n * Pitch + c * 2, 8);
            const size_t at = static_cast<size_t>(n0 + n) * a.y_stride + m0 + c;
            uint16_t *y = static_cast<uint16_t *>(a.y) + at;
            if (m0 + c + 3 < a.M) {
                __builtin_memcpy(y, &w, 8);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (m0 + c + i < a.M) y[i] = static_cast<uint16_t>((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
            }
        }
    }
    template<int Y>
    __device__ __forceinline__ void store(const Fp8LinearArgs &a, const f32x4 (&acc)[TM][TN]) const {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            const int n = n0 + (wc * TN + t) * 16 + (lane & 15);
            if (n >= a.N) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const float v[4] = {acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
                store_rows<Y>(a, n, m0 + (wr * TM + i) * 16 + (lane >> 4) * 4, v);
            }
        }
    }
};

// G groups of WR x WC waves share the tile, group g taking blocks g, g + G, ..
// through a ring of its own; their sums meet in LDS at the end, in group order.
// Y, Sums32: as for k_fp8_split.
template<int WR, int WC, int TM, int TN, int S, int G, bool Tiles, int Y, bool Sums32>
__global__ __launch_bounds__(64 * WR * WC * G) void k_fp8_gemm(Fp8LinearArgs a, int tiles_m) {
    using Tile = GemmTile<WR, WC, TM, TN, S, G, Tiles>;
    constexpr int Sums = TM * TN * Tile::W * 64 * 16;   // bytes of one group's sums
    static_assert(G == 1 || Sums <= G * Tile::Lds);
    static_assert(Sums32 || Y != kF32);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[G][Tile::Lds];
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / Tile::W;
    const Tile g(a, blockIdx.x % tiles_m, blockIdx.x / tiles_m, lds[group]);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int b = 0; b < S - 1; ++b) {
        g.stage_rows(b * G + group, b);
        g.stage_columns(b * G + group, b);
    }
    int at = 0;   // the step's buffer, step % S
    for (int b = group; b - group < a.nb; b += G) {
        // Block b's loads are all but the last S - 2 steps'; memory answers in
        // order, and past the last block a step still issues as many (of scales
        // in fours, most steps load none: Loads counts the fewest).
        wait_for_lds_loads<(S - 2) * Tile::Loads>();
        __syncthreads();
        // Every wave is done with the last step: its buffer takes the one S - 1 ahead.
        const int next = at == 0 ? S - 1 : at - 1;
        g.stage_rows(b + (S - 1) * G, next);
        g.stage_columns(b + (S - 1) * G, next);
        const uint8_t *buf = lds[group] + at * Tile::Buffer;
        at = at + 1 == S ? 0 : at + 1;
        if (G > 1 && b >= a.nb) break;   // the group's share has ended: only the others' barriers were left
        const float sw = g.wscale[b];
        using Operand = std::conditional_t<Sums32, FragF16, Frag>;
        Operand x[TN];
        float s[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            x[t] = operand<Operand>(g.column(buf, t));
            s[t] = g.scale(lds[group], buf, b, t) * sw;
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const Operand w = operand<Operand>(g.row(buf, i));
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const f32x4 p = block_dot(w, x[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(p[e], s[t], acc[i][t][e]);
            }
        }
    }
    wait_for_lds_loads<0>();   // no load may outlive the buffers
    if constexpr (G > 1) {
        f32x4 *sums = reinterpret_cast<f32x4 *>(lds) + g.wave * 64 + g.lane;   // [tile][wave][lane]
#pragma unroll
        for (int q = 1; q < G; ++q) {
            __syncthreads();
            if (group == q) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int t = 0; t < TN; ++t) sums[(i * TN + t) * Tile::W * 64] = acc[i][t];
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int t = 0; t < TN; ++t) acc[i][t] += sums[(i * TN + t) * Tile::W * 64];
            }
        }
        if (group > 0) return;
    }
    if constexpr (G == 1 && Y != kF32) {
        __syncthreads();
        g.template store_along_rows<Y>(a, acc, lds[0]);
    } else {
        g.template store<Y>(a, acc);
    }
}

// The largest batches: 256 x 256 a workgroup, eight waves of 128 x 64, two on
// each SIMD that take turns, one at the MFMAs of half a step (four row tiles
// against four column tiles) while the other reads its next operands from LDS.
// A barrier ends each turn.  With turn p of waves 0 .. 3 at
//   4 b: read columns, rows 0 .. 3 | 4 b + 1: multiply | 4 b + 2: read rows
//   4 .. 7 | 4 b + 3: multiply
// and waves 4 .. 7 one turn behind, block b's buffer is last read in turn 4 b
// + 3; block b + 1's loads start in turns 4 b to 4 b + 2, into the buffer last
// read in turn 4 b - 1, and each wave waits for its own before the barrier
// that ends its second read of block b, turn 4 b + 3 at the latest.
template<bool Tiles, int Y>
__global__ __launch_bounds__(512) void k_fp8_gemm_wide(Fp8LinearArgs a, int tiles_m) {
    using Tile = GemmTile<2, 4, 8, 4, 2, 1, Tiles>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::Lds];
    const Tile g(a, blockIdx.x % tiles_m, blockIdx.x / tiles_m, lds);
    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // Everything issued before it is done and nothing moves across it.
    const auto turn = [](bool loads) {
        __builtin_amdgcn_sched_barrier(0);
        if (loads) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    float s[4];
    g.stage_rows(0, 0);
    g.stage_columns(0, 0);
    turn(true);
    if (g.wr == 1) turn(false);   // waves 4 .. 7: one turn behind
    const auto multiply = [&](const Frag (&w)[4], const Frag (&x)[4], int i0) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 p = block_dot(w[i], x[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i0 + i][t][e] = fmaf(p[e], s[t], acc[i0 + i][t][e]);
            }
        // Four MFMAs ahead, so that no product is waited for.
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
#pragma unroll
        for (int q = 0; q < 12; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);   // VALU
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);   // MFMA
        }
        __builtin_amdgcn_sched_group_barrier(0x2, 16, 0);
        __builtin_amdgcn_s_setprio(0);
    };
    for (int b = 0; b < a.nb; ++b) {
        const uint8_t *buf = lds + (b & 1) * Tile::Buffer;
        const float sw = g.wscale[b];
        Frag x[4], w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = g.column(buf, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = g.row(buf, i);
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t] = g.scale(lds, buf, b, t) * sw;
        __builtin_amdgcn_sched_barrier(0);
        if (b + 1 < a.nb) g.stage_rows(b + 1, (b + 1) & 1);
        turn(false);
        if (b + 1 < a.nb) g.stage_columns(b + 1, (b + 1) & 1);
        multiply(w, x, 0);
        turn(false);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = g.row(buf, 4 + i);
        turn(true);
        multiply(w, x, 4);
        turn(false);
    }
    if (g.wr == 0) turn(false);   // as many turns for every wave
    g.template store_along_rows<Y>(a, acc, lds);
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_fp8_linear {
    int input = 0, output = 0, max_columns = 0, device = 0;
    int nb = 0;
    uint8_t *mem = nullptr;       // tiles, scales
    const float *scales = nullptr;
    uint8_t *ws = nullptr;        // columns as tiles, then scales [nb][columns]
    int sums = MOE_SUMS_AUTO;
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

void release(moe_fp8_linear *L) {
    if (L->mem) (void)hipFree(L->mem);
    if (L->ws) (void)hipFree(L->ws);
    delete L;
}

bool sums32(const moe_fp8_linear *L, int y_type) { return y_type == MOE_F32 || L->sums == MOE_SUMS_F32; }

moe::Fp8LinearArgs base_args(const moe_fp8_linear *L, int columns, void *y, int y_type, int64_t y_stride) {
    moe::Fp8LinearArgs a{};
    a.tiles = L->mem;
    a.wscale = L->scales;
    a.y = y;
    a.y_type = y_type;
    a.y_stride = y_stride;
    a.M = L->output;
    a.N = columns;
    a.K = L->input;
    a.nb = L->nb;
    return a;
}

// Sums32: sums within a block in fp32, for y of any type; else y is of 16 bits.
template<int WR, int WC, int TM, int TN, int S, int G, bool Tiles, bool Sums32>
int launch_gemm(const moe::Fp8LinearArgs &a, hipStream_t s) {
    using Tile = moe::GemmTile<WR, WC, TM, TN, S, G, Tiles>;
    const int tm = (a.M + Tile::BM - 1) / Tile::BM, tn = (a.N + Tile::BN - 1) / Tile::BN;
    const dim3 grid(static_cast<unsigned>(tm) * tn), block(64 * Tile::W * G);
    const auto launch = [&](auto kernel) { kernel<<<grid, block, 0, s>>>(a, tm); };
    if constexpr (Sums32) {
        if (a.y_type == MOE_F32) {
            launch(moe::k_fp8_gemm<WR, WC, TM, TN, S, G, Tiles, moe::kF32, true>);
            return hipGetLastError();
        }
    }
    if (a.y_type == MOE_BF16) launch(moe::k_fp8_gemm<WR, WC, TM, TN, S, G, Tiles, moe::kBF16, Sums32>);
    else launch(moe::k_fp8_gemm<WR, WC, TM, TN, S, G, Tiles, moe::kF16, Sums32>);
    return hipGetLastError();
}

template<int TM, int TN, int W, bool Tiles, bool Sums32>
int launch_split(const moe::Fp8LinearArgs &a, hipStream_t s) {
    const int tm = (a.M + 16 * TM - 1) / (16 * TM), tn = (a.N + 16 * TN - 1) / (16 * TN);
    const dim3 grid(static_cast<unsigned>(tm) * tn), block(64 * W);
    const auto launch = [&](auto kernel) { kernel<<<grid, block, 0, s>>>(a, tm); };
    if constexpr (Sums32) {
        if (a.y_type == MOE_F32) {
            launch(moe::k_fp8_split<TM, TN, W, Tiles, moe::kF32, true>);
            return hipGetLastError();
        }
    }
    if (a.y_type == MOE_BF16) launch(moe::k_fp8_split<TM, TN, W, Tiles, moe::kBF16, Sums32>);
    else launch(moe::k_fp8_split<TM, TN, W, Tiles, moe::kF16, Sums32>);
    return hipGetLastError();
}

template<bool Tiles>
int launch_gemm_wide(const moe::Fp8LinearArgs &a, hipStream_t s) {
    const int tm = (a.M + 255) / 256, tn = (a.N + 255) / 256;
    const dim3 grid(static_cast<unsigned>(tm) * tn), block(512);
    if (a.y_type == MOE_BF16) moe::k_fp8_gemm_wide<Tiles, moe::kBF16><<<grid, block, 0, s>>>(a, tm);
    else moe::k_fp8_gemm_wide<Tiles, moe::kF16><<<grid, block, 0, s>>>(a, tm);
    return hipGetLastError();
}

// LDS of a stream kernel that quantises its columns.
size_t quantize_lds(const moe::Fp8LinearArgs &a) { return static_cast<size_t>(a.N) * a.nb * (moe::kFp8Block + 4); }

// The stream kernel's launch; IN, NT and RT as there.
template<int IN, int NT, int RT>
int launch_stream(const moe::Fp8LinearArgs &a, hipStream_t s) {
    const dim3 grid((a.M + 16 * RT - 1) / (16 * RT), (a.N + 16 * NT - 1) / (16 * NT)), block(64 * std::min(8, a.nb));
    const size_t lds = IN == moe::kCodes || IN == moe::kTiles ? 0 : quantize_lds(a);
    moe::k_fp8_stream<IN, NT, RT><<<grid, block, lds, s>>>(a);
    return hipGetLastError();
}

// The product for quantised columns: canonical rows, or Tiles.
//
// Small products stream the matrix (16 RT rows and 16 NT columns a workgroup, K
// shared out among its waves); beyond that the output tile grows with the
// number of tiles, and where there are few the tile's K is split among waves or
// shared among groups of them.  us for apply (MI355X, launches in a row), with
// bf16 columns, streamed with NT, RT = 1, 1 / 2, 1 / 2, 2 / 2, 4, then as 64 x 64 tiles:
//         2048 x 2048 at 32 / 64:  5.9 / 6.2 / 6.8 / 7.8; 8.3 and
//                                  6.5 / 6.4 / 6.9 / 8.0; 8.6
//         8192 x 8192 at 32 / 64:  22.9 / 16.3 / 15.4 / 17.5; 19.1 and
//                                  40.4 / 26.7 / 22.8 / 18.0; 19.7
//         8192 x 2048 at 100:      16.8 / 14.7 / 12.3 / 15.5; 18.5
// 16-bit results, 64 x 32 split among eight waves / 64 x 64 in two groups / in
// two of half as many waves / 128 x 64 / 128 x 128 / 256 x 256:
//         2048 x 2048 at  256:   8.3 /  9.4 / 10.0 / 12.9 / 16.4 / 29.7
//                         333:  10.0 /  9.7 / 10.3 / 13.3 / 16.7 / 30.1
//                        1000:  15.4 / 15.3 / 12.5 / 14.3 / 18.0 / 30.6
//                        2500:  30.4 / 31.8 / 27.4 / 24.0 / 24.4 / 34.2
//                        3700:  41.4 / 47.4 / 35.5 / 30.7 / 26.9 / 35.5
//         8192 x 8192 at   96:  24.5 / 19.7 / 24.2 / 36.2 / 46.1 / 91.0, streamed 33.7
//                         200:  44.0 / 35.4 / 27.9 / 38.1 / 48.2 / 94.1
//                         700:   133 /   97 /  79  / 73.5 / 74.3 / 111
//                        2048:   331 /  273 /  219 /  187 /  163 / 141
//                        2800 / 3300 / 4300, the last two: 223 / 221, 260 / 244, 327 / 333
//         2048 x 2048 at 7000 / 9000 / 12000, the last two: 46.4 / 45.1, 60.8 / 70.8, 76.1 / 79.5
// fp32, 64 x 32 split among eight waves / 32 x 48 among four / among two / 64 x
// 64 in four groups / in two of half as many waves / 128 x 128 in two groups /
// 128 x 128:
//         2048 x 2048 at  256:   8.7 /  9.8 / 12.1 / 11.7 / 11.9 / 21.6 / 23.3
//                         333:  12.4 / 10.2 / 12.4 / 12.2 / 12.2 / 22.2 / 23.8
//                         700:  16.6 / 14.3 / 14.0 / 19.8 / 15.9 / 22.5 / 24.2
//                        1000:  20.8 / 18.4 / 19.4 / 20.4 / 17.0 / 23.6 / 25.3
//                        1032:  23.3 / 18.2 / 19.3 / 26.4 / 21.8 / 23.4 / 25.1
//                        2000:  36.3 / 29.4 / 28.9 / 35.6 / 28.6 / 26.5 / 28.1
//                        2500:  45.0 / 35.1 / 37.5 / 44.3 / 36.5 / 43.0 / 39.4
//                        3000:  52.8 / 40.2 / 40.7 / 52.1 / 40.4 / 44.0 / 39.7
//         8192 x 8192 at   96:  29.2 / 21.2 / 29.1 / 26.0 / 29.4 / 61.7 / 71.1
//                         128:  29.8 / 30.0 / 31.9 / 26.8 / 30.2 / 63.0 / 73.0
//                         512:   107 /  108 /  95  /  96  /  89  / 78.0 / 83.9
//                         700:   146 /  147 /  132 /  139 /  125 /  128 /  117
// So the larger tiles take what fills the CUs, by how much of their last round of
// 256 tiles is used, and the smaller ones the rest.
template<bool Tiles>
int launch_product(const moe::Fp8LinearArgs &a, bool sums32, hipStream_t s) {
    constexpr int IN = Tiles ? moe::kTiles : moe::kCodes;
    const auto tiles = [&](long m, long n) { return ((a.M + m - 1) / m) * ((a.N + n - 1) / n); };
    if (a.N <= 64 || static_cast<long>(a.M) * a.N <= 320 * 1024) {
        const int row_tiles = (a.M + 15) / 16;
        if (a.N <= 16 || (a.N <= 32 && row_tiles <= 160)) return launch_stream<IN, 1, 1>(a, s);
        if (row_tiles >= 512) return a.N <= 32 ? launch_stream<IN, 2, 2>(a, s) : launch_stream<IN, 2, 4>(a, s);
        return a.N <= 64 ? launch_stream<IN, 2, 1>(a, s) : launch_stream<IN, 2, 2>(a, s);
    }
    const long t64 = tiles(64, 64), t128 = tiles(128, 128), rounds128 = (t128 + 255) / 256;
    if (sums32) {
        if (tiles(64, 32) <= 256) return launch_split<4, 2, 8, Tiles, true>(a, s);
        // The two forms of a number of groups give the same sums, and so do apply
        // and forward.  That has a price: above 256 tiles 32 x 48 among four waves
        // would be faster at some sizes (1,032 columns 18.2 against 19.3, 2,500 35.1
        // against 37.5), but rows have its sums in four groups of 64 x 64 alone (26.4
        // and 44.3 against 21.8 and 36.5).
        const bool fills = t64 <= 512 && 10 * static_cast<long>(a.M) * a.N >= 9 * 4096 * 256 * ((t64 + 255) / 256);
        if (t64 <= 256) {
            if constexpr (Tiles)
                if (!fills) return launch_split<2, 3, 4, true, true>(a, s);
            return launch_gemm<2, 2, 2, 2, 2, 4, Tiles, true>(a, s);
        }
        if (rounds128 > 2 || t128 * 10 >= 256 * rounds128 * (rounds128 == 1 ? 8 : 7))
            return rounds128 == 1 ? launch_gemm<2, 2, 4, 4, 2, 2, Tiles, true>(a, s) : launch_gemm<2, 2, 4, 4, 2, 1, Tiles, true>(a, s);
        if constexpr (Tiles)
            if (!fills) return launch_split<2, 3, 2, true, true>(a, s);
        return launch_gemm<1, 2, 4, 2, 2, 2, Tiles, true>(a, s);
    }
    if (tiles(64, 32) <= 256) return launch_split<4, 2, 8, Tiles, false>(a, s);
    if (t64 <= 256) return launch_gemm<2, 2, 2, 2, 3, 2, Tiles, false>(a, s);
    if (t64 <= 512) return launch_gemm<1, 2, 4, 2, 2, 2, Tiles, false>(a, s);
    if (t128 < 400) return launch_gemm<2, 2, 4, 2, 2, 1, Tiles, false>(a, s);
    const long t256 = tiles(256, 256);
    if (t256 * 5 < 4 * 256 * ((t256 + 255) / 256)) return launch_gemm<2, 2, 4, 4, 2, 1, Tiles, false>(a, s);
    return launch_gemm_wide<Tiles>(a, s);
}

}  // namespace

extern "C" {

int moe_quantize_e4m3(const void *x, int x_type, int64_t x_stride, int width, int columns, void *codes, float *scales,
                      int *error, void *stream) {
    if (width < 1 || width > 16384 || columns < 1 || columns > 65536 || !valid_rows(x, x_type, x_stride, width) || !codes ||
        !aligned(scales, 4) || !aligned(error, 4))
        return kInvalid;
    return moe::launch_quantize_e4m3(x, x_type, x_stride, width, columns, static_cast<uint8_t *>(codes), scales, error,
                                     static_cast<hipStream_t>(stream));
}

int moe_fp8_linear_create(int input, int output, int max_columns, const void *codes, const float *scales,
                          int weights_on_device, int device, moe_fp8_linear **out) {
    if (!out) return kInvalid;
    *out = nullptr;
    if (input < 32 || input > 16384 || input % 32 || output < 1 || output > 262144 || max_columns < 0 || max_columns > 65536 ||
        !codes || !aligned(scales, 4) || device < 0)
        return kInvalid;
    moe::DeviceScope scope(device);
    if (!scope.ok()) return hipErrorInvalidDevice;
    auto *L = new (std::nothrow) moe_fp8_linear;
    if (!L) return hipErrorOutOfMemory;
    L->input = input;
    L->output = output;
    L->max_columns = max_columns;
    L->device = device;
    L->nb = (input + moe::kFp8Block - 1) / moe::kFp8Block;
    const size_t code_bytes = static_cast<size_t>(output) * input;
    const size_t scale_bytes = static_cast<size_t>((output + 127) / 128) * L->nb * 4;
    const auto tile_bytes = [&](int rows) { return static_cast<size_t>((rows + 15) / 16) * L->nb * moe::kFp8TileBytes; };
    const size_t tiles = tile_bytes(output);
    const size_t scale_at = round_up(tiles, 256);
    void *staging = nullptr;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, scale_at + scale_bytes);
    if (r == hipSuccess && max_columns > 0)
        r = hipMalloc(&L->ws, tile_bytes(max_columns) + static_cast<size_t>(L->nb) * max_columns * 4);
    const void *device_codes = codes;
    if (r == hipSuccess && !weights_on_device) {
        r = hipMalloc(&staging, code_bytes);
        if (r == hipSuccess) r = hipMemcpy(staging, codes, code_bytes, hipMemcpyHostToDevice);
        device_codes = staging;
    }
    if (r == hipSuccess) r = moe::launch_fp8_repack(static_cast<const uint8_t *>(device_codes), L->mem, output, input, nullptr);
    if (r == hipSuccess)
        r = hipMemcpy(L->mem + scale_at, scales, scale_bytes, weights_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (staging) (void)hipFree(staging);
    if (r != hipSuccess) { release(L); return r; }
    L->scales = reinterpret_cast<const float *>(L->mem + scale_at);
    *out = L;
    return 0;
}

int moe_fp8_linear_destroy(moe_fp8_linear *L) {
    if (!L) return kInvalid;
    moe::DeviceScope scope(L->device);
    release(L);
    return 0;
}

int moe_fp8_linear_bytes(const moe_fp8_linear *L, size_t *weight_bytes) {
    if (!L || !weight_bytes) return kInvalid;
    *weight_bytes = static_cast<size_t>(L->output) * L->input + static_cast<size_t>((L->output + 127) / 128) * L->nb * 4;
    return 0;
}

int moe_fp8_linear_set_sums(moe_fp8_linear *L, int sums) {
    if (!L || (sums != MOE_SUMS_AUTO && sums != MOE_SUMS_F32)) return kInvalid;
    L->sums = sums;
    return 0;
}

int moe_fp8_linear_forward(moe_fp8_linear *L, const void *x_codes, const float *x_scales, int columns, void *y, int y_type,
                           int64_t y_stride, void *stream) {
    if (!L || !aligned(x_codes, 16) || !aligned(x_scales, 4) || columns < 1 || columns > 65536 ||
        !valid_rows(y, y_type, y_stride, L->output))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    moe::Fp8LinearArgs a = base_args(L, columns, y, y_type, y_stride);
    a.codes = static_cast<const uint8_t *>(x_codes);
    a.xscale = x_scales;
    a.scale_n = L->nb;
    a.scale_b = 1;
    return launch_product<false>(a, sums32(L, y_type), static_cast<hipStream_t>(stream));
}

int moe_fp8_linear_apply(moe_fp8_linear *L, const void *x, int x_type, int64_t x_stride, int columns, void *y, int y_type,
                         int64_t y_stride, int *error, void *stream) {
    if (!L || columns < 1 || columns > L->max_columns || !valid_rows(x, x_type, x_stride, L->input) ||
        !valid_rows(y, y_type, y_stride, L->output) || !aligned(error, 4))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    const auto s = static_cast<hipStream_t>(stream);
    moe::Fp8LinearArgs a = base_args(L, columns, y, y_type, y_stride);
    const auto extent = [&](int64_t stride, int width, int type) {
        return (static_cast<size_t>(columns - 1) * stride + width) * moe::elem_bytes(type);
    };
    const char *xb = static_cast<const char *>(x), *yb = static_cast<const char *>(y);
    const bool apart = xb + extent(x_stride, L->input, x_type) <= yb || yb + extent(y_stride, L->output, y_type) <= xb;
    // Every workgroup (16 rows) quantises all of the columns: in its own kernel
    // where that is up to four passes of its threads, or two where a CU takes
    // more than one workgroup (us, in the product's kernel / in two launches:
    // 2048 x 2048 at 1, 4, 8, 16 columns 3.6 / 5.7, 4.4 / 5.6, 5.5 / 5.7, 7.7 /
    // 5.8; 8192 x 8192 at 1, 2 14.2 / 14.4, 16.5 / 14.4; rows of 2,048 of 8,192
    // at 4, 8 6.0 / 6.3, 7.7 / 6.3).
    if (columns <= 16 && apart && columns * L->nb <= (L->output <= 4096 ? 128 : 64)) {
        a.x = x;
        a.x_stride = x_stride;
        a.error = error;
        if (x_type == MOE_F32) return launch_stream<moe::kF32, 1, 1>(a, s);
        if (x_type == MOE_BF16) return launch_stream<moe::kBF16, 1, 1>(a, s);
        return launch_stream<moe::kF16, 1, 1>(a, s);
    }
    auto *scales = reinterpret_cast<float *>(L->ws + static_cast<size_t>((columns + 15) / 16) * L->nb * moe::kFp8TileBytes);
    const hipError_t r = moe::launch_quantize<true>(x, x_type, x_stride, L->input, columns, L->ws, scales, columns,
                                                    error, s);
    if (r != hipSuccess) return r;
    a.codes = L->ws;
    a.xscale = scales;
    a.scale_n = 1;
    a.scale_b = columns;
    return launch_product<true>(a, sums32(L, y_type), s);
}

}  // extern "C"
