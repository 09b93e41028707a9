// Matrices of e4m3 values with one fp32 scale per block of 128 x 128
// (moe_fp8_linear_*) and the quantiser of their activations:
//   y[n][m] = sum_b sx[n][b] sw[m / 128][b] sum_{k in block b} cx[n][k] cw[m][k]
// The inner sum is one MFMA tile step; its result is multiplied by both
// scales into an fp32 accumulator, and y is rounded once.
#include "moe_ffn.h"
#include "moe_fp8.hpp"

#include <algorithm>
#include <new>

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
// 16 lanes per group of 128, 8 elements each; memory bound.
template<int T>
__global__ __launch_bounds__(256) void k_quantize_e4m3(const void *__restrict__ x, int64_t stride, int width, int nb,
                                                       size_t groups, bool vec, uint8_t *__restrict__ codes,
                                                       float *__restrict__ scales, int *error) {
    const size_t g = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;
    if (g >= groups) return;   // whole groups of 16 lanes
    const int part = threadIdx.x & 15;
    const size_t n = g / nb;
    const int k = static_cast<int>(g % nb) * kFp8Block + part * 8;
    const size_t at = n * static_cast<size_t>(stride) + k;
    float v[8];
    if (vec) {
        Raw8 raw{};
        if (k < width) raw = load8_raw<T>(x, at);
        unpack8<T>(raw, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < width ? load1<T>(x, at + i) : 0.0f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
    m = max(m, static_cast<uint32_t>(lane_xor<1>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<2>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<4>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<8>(static_cast<int>(m))));
    const GroupScale s = group_scale(m);
    uint2 c = make_uint2(pack_e4m3(v[0] * s.r, v[1] * s.r, v[2] * s.r, v[3] * s.r),
                         pack_e4m3(v[4] * s.r, v[5] * s.r, v[6] * s.r, v[7] * s.r));
    if (s.bad) c = make_uint2(0u, 0u);
    uint8_t *out = codes + n * width + k;
    if (vec) {
        if (k < width) *reinterpret_cast<uint2 *>(out) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < width) out[i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
    if (part == 0) {
        scales[g] = s.s;
        if (s.bad) atomicOr(error, 1);
    }
}

}  // namespace

hipError_t launch_fp8_repack(const uint8_t *codes, uint8_t *tiles, size_t rows, int cols, hipStream_t s) {
    const int nb = (cols + kFp8Block - 1) / kFp8Block;
    // A grid holds fewer than 2^32 threads: at most 2^30 chunks a launch.
    const size_t rows_at_once = (size_t{1} << 30) / (static_cast<size_t>(nb) * kFp8TileBytes / 16) * kFp8TileRows;
    for (size_t first = 0; first < rows; first += rows_at_once) {
        const size_t n = std::min(rows_at_once, rows - first);
        const size_t chunks = (n + kFp8TileRows - 1) / kFp8TileRows * nb * (kFp8TileBytes / 16);
        k_fp8_repack<<<dim3(static_cast<unsigned>((chunks + 255) / 256)), dim3(256), 0, s>>>(
            codes + first * cols, reinterpret_cast<uint4 *>(tiles + first / kFp8TileRows * nb * kFp8TileBytes), n, cols, nb,
            chunks);
    }
    return hipGetLastError();
}

hipError_t launch_quantize_e4m3(const void *x, int type, int64_t stride, int width, int columns, uint8_t *codes,
                                float *scales, int *error, hipStream_t s) {
    const int nb = (width + kFp8Block - 1) / kFp8Block;
    const size_t groups = static_cast<size_t>(columns) * nb;
    const dim3 grid(static_cast<unsigned>((groups + 15) / 16)), block(256);
    const bool vec = width % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * elem_bytes(type) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(codes) % 8 == 0;
    switch (type) {
    case kF32: k_quantize_e4m3<kF32><<<grid, block, 0, s>>>(x, stride, width, nb, groups, vec, codes, scales, error); break;
    case kBF16: k_quantize_e4m3<kBF16><<<grid, block, 0, s>>>(x, stride, width, nb, groups, vec, codes, scales, error); break;
    default: k_quantize_e4m3<kF16><<<grid, block, 0, s>>>(x, stride, width, nb, groups, vec, codes, scales, error); break;
    }
    return hipGetLastError();
}

namespace {

struct Fp8LinearArgs {
    const uint8_t *tiles;    // [ceil(M/16)][nb] tiles
    const float *wscale;     // [ceil(M/128)][nb]
    const void *x;           // rows of a type (few columns), or unused
    int64_t x_stride;
    const uint8_t *codes;    // [N][K] e4m3 rows
    const float *xscale;     // [N][nb]
    const uint8_t *zero;     // 16 bytes of zeros
    void *y;
    int64_t y_stride;
    int y_type;
    int y_vec;               // rows of y take 4-element stores
    int x_vec;               // rows of x take 8-element loads
    int M, N, K, nb;
    int *error;
};

// Four results of one token, rows m .. m + 3.
__device__ __forceinline__ void store_rows(const Fp8LinearArgs &a, int n, int m, const float (&v)[4]) {
    const size_t at = static_cast<size_t>(n) * a.y_stride + m;
    if (a.y_vec && m + 3 < a.M) {
        if (a.y_type == kF32) store4<kF32>(a.y, at, v);
        else if (a.y_type == kBF16) store4<kBF16>(a.y, at, v);
        else store4<kF16>(a.y, at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (m + i >= a.M) break;
        if (a.y_type == kF32) store1<kF32>(a.y, at + i, v[i]);
        else if (a.y_type == kBF16) store1<kBF16>(a.y, at + i, v[i]);
        else store1<kF16>(a.y, at + i, v[i]);
    }
}

// A token's 32 elements at k as its fragment, quantised here: the four lanes
// l, l ^ 16, l ^ 32, l ^ 48 hold the token's block.  Elements past the row's
// end count as zero.
template<int T>
__device__ __forceinline__ Frag quantize_frag(const Fp8LinearArgs &a, int n, int k, float &scale, int &flags) {
    const size_t at = static_cast<size_t>(n) * a.x_stride + k;
    const bool in = k < a.K;
    float v[32];
    if (a.x_vec) {
        Raw8 raw[4] = {};
        if (in) {
#pragma unroll
            for (int q = 0; q < 4; ++q) raw[q] = load8_raw<T>(a.x, at + 8 * q);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float u[8];
            unpack8<T>(raw[q], u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * q + i] = u[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = in ? load1<T>(a.x, at + i) : 0.0f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max(m, magnitude(v[i]));
    m = max(m, static_cast<uint32_t>(lane_xor<16>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<32>(static_cast<int>(m))));
    const GroupScale s = group_scale(m);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w[i] = pack_e4m3(v[4 * i] * s.r, v[4 * i + 1] * s.r, v[4 * i + 2] * s.r, v[4 * i + 3] * s.r);
        if (s.bad) w[i] = 0u;
    }
    if (s.bad) flags |= 1;
    scale = s.s;
    return Frag{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}

// Few columns: a workgroup takes 16 rows and 16 NT columns, its waves share
// out the blocks of the row (wave w: blocks w, w + W, ..) and add up through
// LDS in wave order.  The matrix streams from memory straight into registers,
// each tile once per column tile group.
// IN: the columns' type, quantised here (NT = 1), or kCodes.
template<int IN, int NT>
__global__ __launch_bounds__(512) void k_fp8_stream(Fp8LinearArgs a) {
    __shared__ f32x4 red[8][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int W = blockDim.x >> 6, mt = blockIdx.x, n0 = blockIdx.y * 16 * NT;
    const uint8_t *row = a.tiles + static_cast<size_t>(mt) * a.nb * kFp8TileBytes;
    const float *wscale = a.wscale + static_cast<size_t>(mt * kFp8TileRows / kFp8Block) * a.nb;
    const int kl = (lane >> 4) * 32;
    int token[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) token[t] = min(n0 + 16 * t + (lane & 15), a.N - 1);
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int flags = 0;
    constexpr int U = NT == 1 ? 4 : 2;   // blocks whose loads are in flight together
    for (int b0 = wave; b0 < a.nb; b0 += W * U) {
        Frag w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Past the last block: the first one of the round again, with a scale of 0 below.
            const int b = b0 + u * W < a.nb ? b0 + u * W : b0;
            w[u] = load_tile(row + static_cast<size_t>(b) * kFp8TileBytes, lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = b0 + u * W < a.nb;
            if (!in) break;
            const int b = b0 + u * W;
            const FragF16 wf = to_f16(w[u]);
            const float sw = wscale[b];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                Frag x;
                float sx;
                if constexpr (IN == kCodes) {
                    const int k = b * kFp8Block + kl;
                    x = Frag{};
                    if (k < a.K) {
                        const uint4 *p = reinterpret_cast<const uint4 *>(a.codes + static_cast<size_t>(token[t]) * a.K + k);
                        x = Frag{p[0], p[1]};
                    }
                    sx = a.xscale[static_cast<size_t>(token[t]) * a.nb + b];
                } else {
                    x = quantize_frag<IN>(a, token[t], b * kFp8Block + kl, sx, flags);
                }
                const f32x4 p = block_dot(wf, to_f16(x));
                const float s = sx * sw;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(p[i], s, acc[t][i]);
            }
        }
    }
    if constexpr (IN != kCodes) {
        if (mt == 0 && flags) atomicOr(a.error, flags);   // every row tile quantises the same columns
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * NT; i += blockDim.x) {
        const int t = i >> 6, l = i & 63;
        f32x4 s = red[0][t][l];
        for (int q = 1; q < W; ++q) {
            const f32x4 v = red[q][t][l];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = s[e] + v[e];
        }
        const int n = n0 + 16 * t + (l & 15);
        const float v[4] = {s[0], s[1], s[2], s[3]};
        if (n < a.N) store_rows(a, n, mt * kFp8TileRows + (l >> 4) * 4, v);
    }
}

// Many columns: a workgroup of WR x WC waves takes 16 TM WR rows and 16 TN WC
// columns, and steps through the blocks of K with both operands' next step on
// the way to LDS (two buffers) while it multiplies the current one.
template<int WR, int WC, int TM, int TN, bool F16>
__global__ __launch_bounds__(64 * WR * WC) void k_fp8_gemm(Fp8LinearArgs a, int tiles_m, int tiles_n) {
    constexpr int W = WR * WC, BM = 16 * TM * WR, BN = 16 * TN * WC;
    static_assert(kFp8Block % (16 * TM) == 0, "a wave's rows share one scale block");
    constexpr int ABytes = BM * kFp8Block, BBytes = BN * kFp8Block;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][ABytes + BBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    const int pm = blockIdx.x % tiles_m, pn = blockIdx.x / tiles_m;
    const int m0 = pm * BM, n0 = pn * BN, row_tiles = (a.M + 15) / 16;

    // Staging, 1 KiB (64 lanes x 16 bytes) a load.  Rows of the matrix past
    // its end and columns past N read the last one again; they are not stored.
    // Columns: 8 rows of 128 bytes a load, each row's eight chunks permuted by
    // its index so that the fragment reads below spread over the LDS banks.
    constexpr int ALoads = BM / 8, BLoads = BN / 8;
    static_assert(ALoads % W == 0 && BLoads % W == 0, "every wave issues the same number of loads");
    const uint8_t *ap[ALoads / W];
    const uint8_t *bp[BLoads / W];
    int bk[BLoads / W];
#pragma unroll
    for (int i = 0; i < ALoads / W; ++i) {
        const int c = i * W + wave;
        const int tile = min(m0 / 16 + (c >> 1), row_tiles - 1);
        ap[i] = a.tiles + static_cast<size_t>(tile) * a.nb * kFp8TileBytes + (c & 1) * 1024 + lane * 16;
    }
#pragma unroll
    for (int i = 0; i < BLoads / W; ++i) {
        const int c = i * W + wave, t = lane >> 3;
        bk[i] = ((lane & 7) ^ t ^ (c & 1)) * 16;
        bp[i] = a.codes + static_cast<size_t>(min(n0 + 8 * c + t, a.N - 1)) * a.K + bk[i];
    }
    auto stage = [&](int b, uint8_t *buf) {
#pragma unroll
        for (int i = 0; i < ALoads / W; ++i)
            load_to_lds(ap[i] + static_cast<size_t>(b) * kFp8TileBytes, buf + (i * W + wave) * 1024);
#pragma unroll
        for (int i = 0; i < BLoads / W; ++i) {
            const uint8_t *p = b * kFp8Block + bk[i] < a.K ? bp[i] + b * kFp8Block : a.zero;
            load_to_lds(p, buf + ABytes + (i * W + wave) * 1024);
        }
    };

    const float *wscale = a.wscale + static_cast<size_t>(min(m0 + wr * 16 * TM, a.M - 1) / kFp8Block) * a.nb;
    const float *xs[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t)
        xs[t] = a.xscale + static_cast<size_t>(min(n0 + (wc * TN + t) * 16 + (lane & 15), a.N - 1)) * a.nb;
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < TN; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // Fragment of column l % 16, chunks 2 (l / 16) and + 1, in the permuted order.
    const int tok = lane & 15, swz = (tok & 7) ^ (tok >> 3);
    const int boff = (tok >> 3) * 1024 + (tok & 7) * 128;
    const int b0off = boff + (((lane >> 4) * 2) ^ swz) * 16, b1off = boff + (((lane >> 4) * 2 + 1) ^ swz) * 16;

    stage(0, lds[0]);
    for (int b = 0; b < a.nb; ++b) {
        __syncthreads();
        uint8_t *buf = lds[b & 1];
        const float sw = wscale[b];
        float s[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) s[t] = xs[t][b] * sw;
        if (b + 1 < a.nb) stage(b + 1, lds[(b + 1) & 1]);
        const uint8_t *bb = buf + ABytes + wc * TN * 2048;
        Frag x[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t)
            x[t] = Frag{*reinterpret_cast<const uint4 *>(bb + t * 2048 + b0off), *reinterpret_cast<const uint4 *>(bb + t * 2048 + b1off)};
        const uint8_t *ab = buf + wr * TM * 2048;
        if constexpr (F16) {
            FragF16 xf[TN];
#pragma unroll
            for (int t = 0; t < TN; ++t) xf[t] = to_f16(x[t]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const FragF16 w = to_f16(load_tile(ab + i * 2048, lane));
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    const f32x4 p = block_dot(w, xf[t]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(p[e], s[t], acc[i][t][e]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const Frag w = load_tile(ab + i * 2048, lane);
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    const f32x4 p = block_dot(w, x[t]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(p[e], s[t], acc[i][t][e]);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        const int n = n0 + (wc * TN + t) * 16 + (lane & 15);
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const float v[4] = {acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
            store_rows(a, n, m0 + (wr * TM + i) * 16 + (lane >> 4) * 4, v);
        }
    }
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_fp8_linear {
    int input = 0, output = 0, max_columns = 0, device = 0;
    int nb = 0;
    uint8_t *mem = nullptr;       // tiles, scales, 16 bytes of zeros
    const float *scales = nullptr;
    const uint8_t *zero = nullptr;
    uint8_t *ws = nullptr;        // codes [max_columns][input], then scales [max_columns][nb]
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

moe::Fp8LinearArgs base_args(const moe_fp8_linear *L, int columns, void *y, int y_type, int64_t y_stride) {
    moe::Fp8LinearArgs a{};
    a.tiles = L->mem;
    a.wscale = L->scales;
    a.zero = L->zero;
    a.y = y;
    a.y_type = y_type;
    a.y_stride = y_stride;
    const int four = 4 * moe::elem_bytes(y_type);
    a.y_vec = aligned(y, four) && y_stride * moe::elem_bytes(y_type) % four == 0;
    a.M = L->output;
    a.N = columns;
    a.K = L->input;
    a.nb = L->nb;
    return a;
}

template<int WR, int WC, int TM, int TN>
int launch_gemm(const moe::Fp8LinearArgs &a, hipStream_t s) {
    constexpr int BM = 16 * TM * WR, BN = 16 * TN * WC;
    const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    const dim3 grid(static_cast<unsigned>(static_cast<size_t>(tm) * tn)), block(64 * WR * WC);
    if (a.y_type == MOE_F32) moe::k_fp8_gemm<WR, WC, TM, TN, true><<<grid, block, 0, s>>>(a, tm, tn);
    else moe::k_fp8_gemm<WR, WC, TM, TN, false><<<grid, block, 0, s>>>(a, tm, tn);
    return hipGetLastError();
}

// The stream kernel's launch for 16 NT columns a workgroup; IN as there.
template<int IN, int NT>
int launch_stream(const moe::Fp8LinearArgs &a, hipStream_t s) {
    const dim3 grid((a.M + 15) / 16, (a.N + 16 * NT - 1) / (16 * NT)), block(64 * std::min(8, a.nb));
    moe::k_fp8_stream<IN, NT><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

int launch_rows(moe::Fp8LinearArgs a, const uint8_t *codes, const float *scales, hipStream_t s) {
    a.codes = codes;
    a.xscale = scales;
    if (a.N <= 16) return launch_stream<moe::kCodes, 1>(a, s);
    if (a.N <= 32) return launch_stream<moe::kCodes, 2>(a, s);
    if (a.N <= 64) return launch_stream<moe::kCodes, 4>(a, s);
    const long big = static_cast<long>((a.M + 255) / 256) * ((a.N + 255) / 256);
    if (big >= 200) return launch_gemm<2, 4, 8, 4>(a, s);
    const long mid = static_cast<long>((a.M + 127) / 128) * ((a.N + 127) / 128);
    if (mid >= 200) return launch_gemm<2, 2, 4, 4>(a, s);
    return launch_gemm<2, 2, 2, 2>(a, s);
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
    const size_t tiles = static_cast<size_t>((output + 15) / 16) * L->nb * moe::kFp8TileBytes;
    const size_t scale_at = round_up(tiles, 256), zero_at = scale_at + round_up(scale_bytes, 256);
    void *staging = nullptr;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, zero_at + 256);
    if (r == hipSuccess && max_columns > 0)
        r = hipMalloc(&L->ws, static_cast<size_t>(max_columns) * (static_cast<size_t>(input) + L->nb * 4));
    const void *device_codes = codes;
    if (r == hipSuccess && !weights_on_device) {
        r = hipMalloc(&staging, code_bytes);
        if (r == hipSuccess) r = hipMemcpy(staging, codes, code_bytes, hipMemcpyHostToDevice);
        device_codes = staging;
    }
    if (r == hipSuccess) r = moe::launch_fp8_repack(static_cast<const uint8_t *>(device_codes), L->mem, output, input, nullptr);
    if (r == hipSuccess)
        r = hipMemcpy(L->mem + scale_at, scales, scale_bytes, weights_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (r == hipSuccess) r = hipMemset(L->mem + zero_at, 0, 256);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (staging) (void)hipFree(staging);
    if (r != hipSuccess) { release(L); return r; }
    L->scales = reinterpret_cast<const float *>(L->mem + scale_at);
    L->zero = L->mem + zero_at;
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

int moe_fp8_linear_forward(moe_fp8_linear *L, const void *x_codes, const float *x_scales, int columns, void *y, int y_type,
                           int64_t y_stride, void *stream) {
    if (!L || !aligned(x_codes, 16) || !aligned(x_scales, 4) || columns < 1 || columns > 65536 ||
        !valid_rows(y, y_type, y_stride, L->output))
        return kInvalid;
    moe::LaunchDevice device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    return launch_rows(base_args(L, columns, y, y_type, y_stride), static_cast<const uint8_t *>(x_codes), x_scales,
                       static_cast<hipStream_t>(stream));
}

int moe_fp8_linear_apply(moe_fp8_linear *L, const void *x, int x_type, int64_t x_stride, int columns, void *y, int y_type,
                         int64_t y_stride, int *error, void *stream) {
    if (!L || columns < 1 || columns > L->max_columns || !valid_rows(x, x_type, x_stride, L->input) ||
        !valid_rows(y, y_type, y_stride, L->output) || !aligned(error, 4))
        return kInvalid;
    moe::LaunchDevice device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    const auto s = static_cast<hipStream_t>(stream);
    moe::Fp8LinearArgs a = base_args(L, columns, y, y_type, y_stride);
    const auto extent = [&](int64_t stride, int width, int type) {
        return (static_cast<size_t>(columns - 1) * stride + width) * moe::elem_bytes(type);
    };
    const char *xb = static_cast<const char *>(x), *yb = static_cast<const char *>(y);
    const bool apart = xb + extent(x_stride, L->input, x_type) <= yb || yb + extent(y_stride, L->output, y_type) <= xb;
    if (columns <= 16 && apart) {
        a.x = x;
        a.x_stride = x_stride;
        a.x_vec = aligned(x, 16) && x_stride * moe::elem_bytes(x_type) % 16 == 0;
        a.error = error;
        if (x_type == MOE_F32) return launch_stream<moe::kF32, 1>(a, s);
        if (x_type == MOE_BF16) return launch_stream<moe::kBF16, 1>(a, s);
        return launch_stream<moe::kF16, 1>(a, s);
    }
    auto *scales = reinterpret_cast<float *>(L->ws + static_cast<size_t>(L->max_columns) * L->input);
    const hipError_t r = moe::launch_quantize_e4m3(x, x_type, x_stride, L->input, columns, L->ws, scales, error, s);
    if (r != hipSuccess) return r;
    return launch_rows(a, L->ws, scales, s);
}

}  // extern "C"
