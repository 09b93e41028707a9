// A routed-expert layer of e4m3 matrices for a few tokens (moe_fp8_layer_*),
// in two launches:
//   gate_up    per (expert that a token reaches, slice of intermediate rows):
//              the tokens' rows quantised to e4m3, gate and up products, SiLU(g) u
//   down_fold  per (token, slice of output rows): each rank's middle row
//              quantised, its down product, and the weighted sum in rank order
//              with the shared expert
// Both are bound by the experts' bytes (6 H I flops a token and expert against
// 3 H I bytes an expert).  gate_up reads every byte of a reached expert once
// however many tokens share it; down_fold reads an expert's rows for each of
// its tokens, by workgroups of one XCD at about the same time, so that its L2
// serves all but the first.
#include "moe_ffn.h"
#include "moe_fp8.hpp"

#include <algorithm>
#include <climits>
#include <cstdlib>
#include <new>

namespace moe {

inline constexpr int kFp8LayerTokens = 64;   // tokens of one forward: a lane each in the grouping

namespace {

struct Fp8LayerArgs {
    const uint8_t *gate, *up, *down;           // tiles [E'][rows/16][blocks]
    const float *gate_s, *up_s, *down_s;       // [E'][ceil(rows/128)][blocks]
    const void *x;             // [T][H]
    const int32_t *ids;        // [T][k]
    const float *weights;      // [T][k]
    const float *shared_gate;  // [T] or null
    float *middle;             // [T][P1][I] fp32 SiLU(g) u
    void *y;                   // [T][H]
    int *error;
    int T, H, I, E, k, P1;     // P1 = k + shared
    int nbh, nbi;
};

inline constexpr int kTileWaves = 4, kRowTiles = 8 / kTileWaves;   // waves of a row tile, row tiles of a gate_up item
static_assert(32 % (16 * kRowTiles) == 0, "the intermediate size is a multiple of 32");
inline constexpr int kGateUpGroups = 512;   // workgroups of gate_up: two a CU
inline constexpr int kChunk = 24;   // blocks of K whose columns a workgroup holds in LDS: 50 KB

// The routes of the batch, in the registers of a workgroup of 512 threads:
// thread i holds ids i, i + 512, .. (-1 past the last, and for bad ids).
struct Routes {
    static constexpr int Own = kFp8LayerTokens * 32 / 512;
    int id[Own];
    __device__ __forceinline__ explicit Routes(const Fp8LayerArgs &a) {
        const int routes = a.T * a.k;
#pragma unroll
        for (int i = 0; i < Own; ++i) {
            const int q = threadIdx.x + i * 512;
            const int e = q < routes ? a.ids[q] : -1;
            id[i] = e < a.E ? e : -1;
        }
    }
};

// The experts that the batch reaches, each once: the shared expert, then the
// others in the order of their first routes.  Returns their number.
// first [E]: scratch in LDS; list: up to 1 + T k.
__device__ __forceinline__ int list_experts(const Fp8LayerArgs &a, const Routes &q, int *first, int *list) {
    __shared__ int counts[Routes::Own * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, shared = a.P1 > a.k ? 1 : 0;
    if (a.T * a.k <= 64) {
        // Every wave on its own, a route a lane.
        int mine = lane < a.T * a.k ? a.ids[lane] : -1;
        if (mine >= a.E) mine = -1;
        bool later = mine < 0;
        for (int i = 0; i + 1 < a.T * a.k; ++i) later |= lane > i && mine == __builtin_amdgcn_readlane(mine, i);
        const uint64_t is_first = __builtin_amdgcn_ballot_w64(!later);
        if (wave == 0) {
            if (lane == 0 && shared) list[0] = a.E;
            if (!later) list[shared + __builtin_popcountll(is_first & ((uint64_t{1} << lane) - 1))] = mine;
        }
        __syncthreads();
        return shared + __builtin_popcountll(is_first);
    }
    for (int i = threadIdx.x; i < a.E; i += 512) first[i] = INT_MAX;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Routes::Own; ++i)
        if (q.id[i] >= 0) atomicMin(&first[q.id[i]], static_cast<int>(threadIdx.x) + i * 512);
    __syncthreads();
    uint64_t is_first[Routes::Own];
#pragma unroll
    for (int i = 0; i < Routes::Own; ++i) {
        is_first[i] = __builtin_amdgcn_ballot_w64(q.id[i] >= 0 && first[q.id[i] >= 0 ? q.id[i] : 0] ==
                                                                      static_cast<int>(threadIdx.x) + i * 512);
        if (lane == 0) counts[i * 8 + wave] = __builtin_popcountll(is_first[i]);
    }
    if (threadIdx.x == 0 && shared) list[0] = a.E;
    __syncthreads();
    int before = shared, total = shared;
    for (int i = 0; i < Routes::Own * 8; ++i) total += counts[i];
#pragma unroll
    for (int i = 0; i < Routes::Own; ++i) {
        before = shared;
        for (int j = 0; j < i * 8 + wave; ++j) before += counts[j];
        if (is_first[i] >> lane & 1) list[before + __builtin_popcountll(is_first[i] & ((uint64_t{1} << lane) - 1))] = q.id[i];
    }
    __syncthreads();
    return total;
}

// The tokens of one expert and its rank in each, in token order; a token's
// repeat of an id counts at its first rank.
struct Members {
    int rank_of[kFp8LayerTokens];
    int token[kFp8LayerTokens], rank[kFp8LayerTokens];
    int count;
};
__device__ __forceinline__ int find_members(const Fp8LayerArgs &a, const Routes &q, int e, Members &m) {
    const int lane = threadIdx.x & 63;
    if (a.T == 1) {
        if (threadIdx.x < 64) {
            const uint64_t at = __builtin_amdgcn_ballot_w64(q.id[0] == e);   // e of the batch's own, or the shared one
            if (lane == 0) {
                m.token[0] = 0;
                m.rank[0] = e == a.E ? a.k : __builtin_ctzll(at);
            }
        }
        __syncthreads();
        return 1;
    }
    if (threadIdx.x < kFp8LayerTokens)
        m.rank_of[threadIdx.x] = e == a.E && static_cast<int>(threadIdx.x) < a.T ? a.k : INT_MAX;
    __syncthreads();
    if (e < a.E) {
#pragma unroll
        for (int i = 0; i < Routes::Own; ++i) {
            const int r = threadIdx.x + i * 512;
            if (q.id[i] == e) atomicMin(&m.rank_of[r / a.k], r % a.k);
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int r = m.rank_of[lane];
        const uint64_t in = __builtin_amdgcn_ballot_w64(r != INT_MAX);
        if (r != INT_MAX) {
            const int at = __builtin_popcountll(in & ((uint64_t{1} << lane) - 1));
            m.token[at] = lane;
            m.rank[at] = r;
        }
        if (lane == 0) m.count = __builtin_popcountll(in);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(m.count);
}

// Blocks k0 .. k0 + kb - 1 of `cols` rows of x (row i at rows(i), K elements
// of type T_) as one operand tile a block in LDS, and their scales [block][16].
// 16 threads a block.
template<int T_, class Rows>
__device__ __forceinline__ void quantize_columns(const void *x, Rows rows, int cols, int K, int k0, int kb, uint8_t *tiles,
                                                 float *scales) {
    const int part = threadIdx.x & 15;
    for (int i = threadIdx.x >> 4; i < cols * kb; i += 512 / 16) {
        const int c = i / kb, b = i % kb, col = (k0 + b) * kFp8Block + part * 8;
        Raw8 raw{};
        if (col < K) raw = load8_raw<T_>(x, rows(c) + col);
        float v[8];
        unpack8<T_>(raw, v);
        const GroupScale g = group_scale(max16(v));
        *reinterpret_cast<uint2 *>(tiles + b * kFp8TileBytes + tile_offset(part, c)) = quantize8(v, g);
        if (part == 0) scales[b * 16 + c] = g.s;
    }
}

// ------------------------------------------------------------ gate and up ---
// Work item (expert, s): two tiles of 16 rows, four waves a tile, of which wave
// w multiplies blocks w, w + 4, .. of all of the expert's tokens, 16 at a time;
// the sums meet in LDS, in wave order.  A workgroup lists the experts and takes
// items in turn, each with its first tiles on their way before the last one's
// sums are done.  64 tokens, 2048/512, layer time in us with top-10 of 512
// uniform / Zipf(1.1): 274 / 205 with a workgroup per route and slice, of
// which those of an expert's later routes end at once, 244 / 170 so (235 / 165
// with the down kernel as it is now); with eight or two waves a tile 258 / 191
// and 251 / 178.  Four waves a SIMD (two
// workgroups a CU): with two blocks a round in flight the kernel needs 167
// registers and one fits (268 / 185).
template<int T_>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4))) void k_fp8_gate_up(Fp8LayerArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // column tiles [blocks][2048], scales [blocks][16]; then the sums
    __shared__ Members m;
    __shared__ int list[1 + kFp8LayerTokens * 32];
    constexpr int KW = kTileWaves, RW = kRowTiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, rw = wave / KW;
    const int row_tiles = a.I / 16, S = row_tiles / RW;   // I is a multiple of 32
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        // A token's input flags, whatever becomes of its routes.
        bool bad = false;
        for (int i = threadIdx.x; i < a.H; i += 512) bad |= !isfinite(load1<T_>(a.x, static_cast<size_t>(t) * a.H + i));
        if (bad) atomicOr(a.error, 1);
    }
    const Routes routes(a);
    const int items = list_experts(a, routes, reinterpret_cast<int *>(lds), list) * S;
    Frag gf[2], uf[2];   // a block's, and the next one's on their way
    const uint8_t *gw = a.gate, *uw = a.up;
    // Block k0 + b of an item's tile; past the chunk its last block again, not used.
    auto load = [&](int k0, int kb, int b, Frag &g, Frag &v) {
        const size_t at = static_cast<size_t>(k0 + min(b, kb - 1)) * kFp8TileBytes;
        g = load_tile(gw + at, lane);
        v = load_tile(uw + at, lane);
    };
    auto select = [&](int item) {
        const int e = __builtin_amdgcn_readfirstlane(list[item / S]), tile = item % S * RW + rw;
        const size_t at = (static_cast<size_t>(e) * row_tiles + tile) * a.nbh * kFp8TileBytes;
        gw = a.gate + at;
        uw = a.up + at;
        load(0, min(kChunk, a.nbh), kw, gf[0], uf[0]);
        return e;
    };
    int flags = 0, e = static_cast<int>(blockIdx.x) < items ? select(blockIdx.x) : 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int s = item % S, tile = s * RW + rw;
        const int count = find_members(a, routes, e, m);
        const size_t scale0 = (static_cast<size_t>(e) * ((a.I + kFp8Block - 1) / kFp8Block) + tile * 16 / kFp8Block) * a.nbh;
        const float *gs = a.gate_s + scale0, *us = a.up_s + scale0;
        for (int c0 = 0; c0 < count; c0 += 16) {
            const int cols = min(16, count - c0);
            f32x4 ga = {0.0f, 0.0f, 0.0f, 0.0f}, ua = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int k0 = 0; k0 < a.nbh; k0 += kChunk) {
                const int kb = min(kChunk, a.nbh - k0);
                float *xs = reinterpret_cast<float *>(lds + kb * kFp8TileBytes);
                auto multiply = [&](int b, const Frag &g, const Frag &v) {
                    const FragF16 x = to_f16(load_tile(lds + b * kFp8TileBytes, lane));
                    const float sx = xs[b * 16 + (lane & 15)];
                    const f32x4 gp = block_dot(to_f16(g), x), up = block_dot(to_f16(v), x);
                    const float sg = sx * gs[k0 + b], su = sx * us[k0 + b];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        ga[q] = fmaf(gp[q], sg, ga[q]);
                        ua[q] = fmaf(up[q], su, ua[q]);
                    }
                };
                if (c0 > 0 || k0 > 0) load(k0, kb, kw, gf[0], uf[0]);
                quantize_columns<T_>(a.x, [&](int c) { return static_cast<size_t>(m.token[c0 + c]) * a.H; }, cols, a.H, k0, kb, lds, xs);
                __syncthreads();
                for (int b = kw; b < kb; b += 2 * KW) {
                    if (b + KW < kb) load(k0, kb, b + KW, gf[1], uf[1]);
                    multiply(b, gf[0], uf[0]);
                    if (b + 2 * KW < kb) load(k0, kb, b + 2 * KW, gf[0], uf[0]);
                    if (b + KW < kb) multiply(b + KW, gf[1], uf[1]);
                }
                __syncthreads();   // the columns are used up
            }
            f32x4 *red = reinterpret_cast<f32x4 *>(lds);   // [wave][gate, up][lane]
            red[(wave * 2 + 0) * 64 + lane] = ga;
            red[(wave * 2 + 1) * 64 + lane] = ua;
            if (c0 + 16 >= count && item + static_cast<int>(gridDim.x) < items) e = select(item + gridDim.x);
            __syncthreads();
            // Sum i of a row tile: row 4 (lane / 16) + i % 4 of column lane % 16, lane = i / 4.
            const float *sum = reinterpret_cast<const float *>(lds);
            for (int i = threadIdx.x; i < 256 * RW; i += 512) {
                const int r = i >> 8, j = i & 255, c = (j >> 2) & 15, row = (s * RW + r) * 16 + (j >> 6) * 4 + (j & 3);
                if (c >= cols) continue;
                const float *w = sum + r * KW * 512 + j;
                float g = w[0], u = w[256];
#pragma unroll
                for (int q = 1; q < KW; ++q) {
                    g = g + w[q * 512];
                    u = u + w[q * 512 + 256];
                }
                const size_t pair = static_cast<size_t>(m.token[c0 + c]) * a.P1 + m.rank[c0 + c];
                a.middle[pair * a.I + row] = silu_mul(g, u, flags);
            }
            __syncthreads();   // the sums are used up
        }
    }
    if (flags) atomicOr(a.error, flags);
}

inline constexpr int kMaxPairs = 33;   // 32 routes and the shared expert

// Route r of token t, by a whole wave: its expert (the shared one for r = k),
// -1 for a bad id or a repeat of an earlier rank; its weight or gate.
__device__ __forceinline__ int route(const Fp8LayerArgs &a, int t, int r, float &w, int &flags) {
    if (r == a.k) {
        w = a.shared_gate ? a.shared_gate[t] : 1.0f;
        return a.E;
    }
    const int lane = threadIdx.x & 63;
    const int mine = lane < a.k ? a.ids[t * a.k + lane] : -1;
    w = a.weights[t * a.k + r];
    const int e = __builtin_amdgcn_readlane(mine, r);
    if (!isfinite(w) || w < 0.0f) flags |= 1;
    if (e < 0 || e >= a.E || __builtin_amdgcn_ballot_w64(lane < r && mine == e)) {
        flags |= 1;
        return -1;
    }
    return e;
}

// ------------------------------------------------------- down and the sum ---
// Workgroup (t, slice of 16 `tiles` rows); wave w takes ranks w, w + W, ..  It
// quantises the rank's middle row in pieces of eight blocks and streams the
// expert's row tiles past it, U blocks a round with the next round's loads on
// their way.  All 16 columns of its MFMA hold the one token, so every lane has
// its results.
// Six waves a SIMD: two workgroups of eleven waves (top-10 and the shared
// expert) fit a CU, one streaming while the other starts or sums up.  2048/512,
// 1 / 8 / 64 tokens 6.1 / 19.6 / 65 us: bound by latency, then by HBM (79 MB at
// 4.0 TB/s), then by the tiles' way from L2 (720 MB) and their conversions.  The
// middle's codes lie in LDS as fp16 already: widened again for every row tile,
// they were half of the conversions (6.9 / 20.7 / 67).
inline constexpr int kDownPiece = 8, kDownTiles = 16;
template<int T_>
__global__ __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(6))) void k_fp8_down_fold(Fp8LayerArgs a, int tiles) {
    extern __shared__ __attribute__((aligned(16))) float part[];   // [rank][16 tiles]
    __shared__ __attribute__((aligned(16))) _Float16 codes[16][kDownPiece * kFp8Block];   // widened, once for all of the rows
    __shared__ float scales[16][kDownPiece];
    constexpr int U = 2;
    const int R = 16 * tiles;
    __shared__ float weight[kMaxPairs];
    __shared__ int valid[kMaxPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    // Workgroup i runs on XCD i % 8: all tokens of one slice on one XCD, one
    // after the other, so that experts they share come from its L2.
    const int row_tiles = a.H / 16, S = (row_tiles + tiles - 1) / tiles;
    const int j = blockIdx.x >> 3, t = j % a.T, s = (blockIdx.x & 7) + 8 * (j / a.T);
    if (s >= S) return;
    const int tile0 = s * tiles, here = min(tiles, row_tiles - tile0);   // this slice's tiles
    int flags = 0;
    for (int r = wave; r < a.P1; r += W) {
        float w;
        const int e = route(a, t, r, w, flags);
        if (lane == 0) {
            weight[r] = w;
            valid[r] = e >= 0;
        }
        if (e < 0) continue;
        const uint8_t *dw = a.down + (static_cast<size_t>(e) * row_tiles + tile0) * a.nbi * kFp8TileBytes;
        const float *ds = a.down_s + static_cast<size_t>(e) * ((a.H + kFp8Block - 1) / kFp8Block) * a.nbi;
        const float *mid = a.middle + (static_cast<size_t>(t) * a.P1 + r) * a.I;
        for (int k0 = 0; k0 < a.nbi; k0 += kDownPiece) {
            const int kb = min(kDownPiece, a.nbi - k0), rounds = (kb + U - 1) / U, n1 = here * rounds;
            Frag wf[2][U];
            // Round n: tile n / rounds, blocks U (n % rounds) .. of the piece.
            const auto load = [&](int n, Frag (&f)[U]) {
                const size_t tile = min(n / rounds, here - 1);
#pragma unroll
                for (int u = 0; u < U; ++u)   // past the piece: its last block again, not used
                    f[u] = load_tile(dw + (tile * a.nbi + k0 + min(n % rounds * U + u, kb - 1)) * kFp8TileBytes, lane);
            };
            load(0, wf[0]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last piece's reads are done
#pragma unroll
            for (int h = 0; h < kDownPiece / 4; ++h) {
                // Lane l: elements 8 l .. + 7 of 512.
                const int col = (k0 + 4 * h) * kFp8Block + lane * 8;
                if (4 * h >= kb) break;
                Raw8 raw{};
                if (col < a.I) raw = load8_raw<kF32>(mid, col);
                float v[8];
                unpack8<kF32>(raw, v);
                const GroupScale g = group_scale(max16(v));
                const uint2 c = quantize8(v, g);
                *reinterpret_cast<f16x8 *>(&codes[wave][h * 512 + lane * 8]) = e4m3_to_f16(c.x, c.y);
                if ((lane & 15) == 0) scales[wave][4 * h + (lane >> 4)] = g.s;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            f32x4 acc;
            const auto multiply = [&](int n, const Frag (&f)[U]) {
                const int tile = n / rounds, q = n % rounds;
                const float *sw = ds + (tile0 + tile) * 16 / kFp8Block * a.nbi + k0;
                f32x4 *out = reinterpret_cast<f32x4 *>(&part[r * R + 16 * tile + (lane >> 4) * 4]);
                if (q == 0) acc = k0 > 0 ? *out : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int b = q * U + u;
                    if (b >= kb) break;
                    const f16x8 *c = reinterpret_cast<const f16x8 *>(&codes[wave][b * kFp8Block + (lane >> 4) * 32]);
                    const f32x4 p = block_dot(to_f16(f[u]), FragF16{{c[0], c[1], c[2], c[3]}});
                    const float sc = scales[wave][b] * sw[b];
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] = fmaf(p[i], sc, acc[i]);
                }
                if (q == rounds - 1 && (lane & 15) == 0) *out = acc;
            };
            for (int n = 0; n < n1; n += 2) {
                load(n + 1, wf[1]);
                multiply(n, wf[0]);
                if (n + 1 >= n1) break;
                load(n + 2, wf[0]);
                multiply(n + 1, wf[1]);
            }
        }
    }
    if (s == 0 && flags && lane == 0) atomicOr(a.error, flags);
    __syncthreads();
    for (int row = threadIdx.x; row < here * 16; row += blockDim.x) {
        int f = 0;
        const float v = fold(a.k, a.P1 > a.k, a.shared_gate != nullptr, valid, weight, [&](int r) { return part[r * R + row]; }, f);
        store1<T_>(a.y, static_cast<size_t>(t) * a.H + tile0 * 16 + row, v);
        if (f) atomicOr(a.error, f);
    }
}

size_t column_bytes(int blocks) { return static_cast<size_t>(std::min(blocks, kChunk)) * (kFp8TileBytes + 64); }

template<int T_>
hipError_t launch_gate_up(const Fp8LayerArgs &a, hipStream_t s) {
    const int experts = std::min(a.T * a.k, a.E) + (a.P1 > a.k ? 1 : 0);   // at most
    const int slices = a.I / 16 / kRowTiles, grid = std::min(experts * slices, kGateUpGroups);
    const size_t lds = std::max({column_bytes(a.nbh), size_t{8 * 2048}, static_cast<size_t>(a.E) * 4});
    k_fp8_gate_up<T_><<<dim3(grid), dim3(512), lds, s>>>(a);
    return hipGetLastError();
}

template<int T_>
hipError_t launch_layer(const Fp8LayerArgs &a, hipStream_t s) {
    const hipError_t r = launch_gate_up<T_>(a, s);
    if (r != hipSuccess) return r;
    const int row_tiles = a.H / 16;
    // Row tiles a workgroup: the fewest on the busiest CU, and of such choices
    // one workgroup a CU for few tokens, two (which fit at once) for more: us a
    // layer of 2048/512 with 2 / 4 / 8 / 16, 8 tokens 53.7 / 52.7 / 60.6 / 80.3,
    // 32 tokens 166 / 157 / 151 / 155, 64 tokens 271 / 253 / 249 / 235.
    int tiles = 1, best = INT_MAX, best_off = 0;
    for (int n = 1; n <= kDownTiles; ++n) {
        const int rounds = (a.T * ((row_tiles + n - 1) / n) + 255) / 256, off = std::abs(rounds - (a.T <= 8 ? 1 : 2));
        if (rounds * n < best || (rounds * n == best && off < best_off)) {
            tiles = n;
            best = rounds * n;
            best_off = off;
        }
    }
    const dim3 grid(static_cast<unsigned>((row_tiles + tiles - 1) / tiles + 7) / 8 * 8 * a.T), block(64 * std::min(16, a.P1));
    k_fp8_down_fold<T_><<<grid, block, static_cast<size_t>(a.P1) * tiles * 64, s>>>(a, tiles);
    return hipGetLastError();
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_fp8_layer {
    moe_fp8_layer_config cfg{};
    int device = 0;
    uint8_t *mem = nullptr;      // gate, up, down tiles; their scales
    float *middle = nullptr;
    moe::Fp8LayerArgs args{};    // what does not change from call to call
};

namespace {

constexpr int kInvalid = hipErrorInvalidValue;

bool aligned(const void *p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }
int blocks(int n) { return (n + moe::kFp8Block - 1) / moe::kFp8Block; }

bool valid_config(const moe_fp8_layer_config *c) {
    return c && c->hidden >= 32 && c->hidden <= 16384 && c->hidden % 32 == 0 && c->intermediate >= 32 &&
           c->intermediate <= 16384 && c->intermediate % 32 == 0 && c->experts >= 1 && c->experts <= 4096 && c->top_k >= 1 &&
           c->top_k <= 32 && c->top_k <= c->experts && (c->has_shared == 0 || c->has_shared == 1) && c->max_tokens >= 1 &&
           c->max_tokens <= moe::kFp8LayerTokens;
}

// One of the three matrices of every expert: sizes and where its parts lie.
struct Part {
    int rows, cols;
    size_t tiles, scales;            // per expert: bytes of tiles, number of scales
    size_t tiles_at, scales_at;      // byte offsets of expert 0
};
size_t layout(const moe_fp8_layer_config &c, Part (&p)[3]) {
    const int H = c.hidden, I = c.intermediate;
    const size_t Ep = static_cast<size_t>(c.experts) + c.has_shared;
    size_t at = 0;
    for (int i = 0; i < 3; ++i) {
        p[i].rows = i == 2 ? H : I;
        p[i].cols = i == 2 ? I : H;
        p[i].tiles = static_cast<size_t>(p[i].rows / moe::kFp8TileRows) * blocks(p[i].cols) * moe::kFp8TileBytes;
        p[i].scales = static_cast<size_t>(blocks(p[i].rows)) * blocks(p[i].cols);
        p[i].tiles_at = at;
        at += round_up(p[i].tiles * Ep, 256);
    }
    for (int i = 0; i < 3; ++i) {
        p[i].scales_at = at;
        at += round_up(p[i].scales * Ep * 4, 256);
    }
    return at;
}

void release(moe_fp8_layer *L) {
    if (L->mem) (void)hipFree(L->mem);
    if (L->middle) (void)hipFree(L->middle);
    delete L;
}

// `count` experts' matrices from expert `first` on.
hipError_t upload(moe_fp8_layer *L, const Part &p, const moe_fp8_matrix &m, size_t first, size_t count, bool on_device) {
    const size_t bytes = count * p.rows * p.cols;
    const void *codes = m.codes;
    void *staging = nullptr;
    hipError_t r = hipSuccess;
    if (!on_device) {
        if ((r = hipMalloc(&staging, bytes)) != hipSuccess) return r;
        r = hipMemcpy(staging, m.codes, bytes, hipMemcpyHostToDevice);
        codes = staging;
    }
    if (r == hipSuccess)
        r = moe::launch_fp8_repack(static_cast<const uint8_t *>(codes), L->mem + p.tiles_at + first * p.tiles, count * p.rows,
                                   p.cols, nullptr);
    if (r == hipSuccess)
        r = hipMemcpy(L->mem + p.scales_at + first * p.scales * 4, m.scales, count * p.scales * 4,
                      on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (staging) (void)hipFree(staging);
    return r;
}

}  // namespace

extern "C" {

int moe_fp8_layer_memory_bytes(const moe_fp8_layer_config *c, size_t *weight_bytes, size_t *workspace_bytes) {
    if (!valid_config(c) || !weight_bytes || !workspace_bytes) return kInvalid;
    Part p[3];
    *weight_bytes = layout(*c, p);
    *workspace_bytes = static_cast<size_t>(c->max_tokens) * (c->top_k + c->has_shared) * c->intermediate * 4;
    return 0;
}

int moe_fp8_layer_create(const moe_fp8_layer_config *c, const moe_fp8_matrix *experts, const moe_fp8_matrix *shared,
                         int weights_on_device, int device, moe_fp8_layer **out) {
    if (!out) return kInvalid;
    *out = nullptr;
    if (!valid_config(c) || !experts || (c->has_shared && !shared) || device < 0) return kInvalid;
    for (int i = 0; i < 3; ++i) {
        if (!experts[i].codes || !aligned(experts[i].scales, 4)) return kInvalid;
        if (c->has_shared && (!shared[i].codes || !aligned(shared[i].scales, 4))) return kInvalid;
    }
    moe::DeviceScope scope(device);
    if (!scope.ok()) return hipErrorInvalidDevice;
    auto *L = new (std::nothrow) moe_fp8_layer;
    if (!L) return hipErrorOutOfMemory;
    L->cfg = *c;
    L->device = device;
    Part p[3];
    size_t weight_bytes = 0, workspace_bytes = 0;
    (void)moe_fp8_layer_memory_bytes(c, &weight_bytes, &workspace_bytes);
    (void)layout(*c, p);
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, weight_bytes);
    if (r == hipSuccess) r = hipMalloc(&L->middle, workspace_bytes);
    for (int i = 0; i < 3 && r == hipSuccess; ++i) {
        r = upload(L, p[i], experts[i], 0, c->experts, weights_on_device != 0);
        if (r == hipSuccess && c->has_shared) r = upload(L, p[i], shared[i], c->experts, 1, weights_on_device != 0);
    }
    if (r != hipSuccess) { release(L); return r; }
    moe::Fp8LayerArgs &a = L->args;
    a.gate = L->mem + p[0].tiles_at;
    a.up = L->mem + p[1].tiles_at;
    a.down = L->mem + p[2].tiles_at;
    a.gate_s = reinterpret_cast<const float *>(L->mem + p[0].scales_at);
    a.up_s = reinterpret_cast<const float *>(L->mem + p[1].scales_at);
    a.down_s = reinterpret_cast<const float *>(L->mem + p[2].scales_at);
    a.middle = L->middle;
    a.H = c->hidden;
    a.I = c->intermediate;
    a.E = c->experts;
    a.k = c->top_k;
    a.P1 = c->top_k + c->has_shared;
    a.nbh = blocks(c->hidden);
    a.nbi = blocks(c->intermediate);
    *out = L;
    return 0;
}

int moe_fp8_layer_destroy(moe_fp8_layer *L) {
    if (!L) return kInvalid;
    moe::DeviceScope scope(L->device);
    release(L);
    return 0;
}

int moe_fp8_layer_forward(moe_fp8_layer *L, const void *x, int type, const int32_t *ids, const float *weights, int tokens,
                          const float *shared_gate, void *y, int *error, void *stream) {
    if (!L || (type != MOE_F32 && type != MOE_BF16 && type != MOE_F16) || tokens < 1 || tokens > L->cfg.max_tokens ||
        !aligned(x, 16) || !aligned(ids, 4) || !aligned(weights, 4) || (shared_gate && !aligned(shared_gate, 4)) ||
        !aligned(y, moe::elem_bytes(type)) || !aligned(error, 4))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    moe::Fp8LayerArgs a = L->args;
    a.x = x;
    a.ids = ids;
    a.weights = weights;
    a.shared_gate = shared_gate;
    a.y = y;
    a.error = error;
    a.T = tokens;
    const auto s = static_cast<hipStream_t>(stream);
    if (type == MOE_F32) return moe::launch_layer<moe::kF32>(a, s);
    if (type == MOE_BF16) return moe::launch_layer<moe::kBF16>(a, s);
    return moe::launch_layer<moe::kF16>(a, s);
}

}  // extern "C"
