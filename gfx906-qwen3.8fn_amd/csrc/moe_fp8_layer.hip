// A routed-expert layer of e4m3 matrices for a few tokens (moe_fp8_layer_*),
// in two launches:
//   gate_up    per (expert that a token reaches, 16 intermediate rows): the
//              tokens' rows quantised to e4m3, gate and up products, SiLU(g) u
//   down_fold  per (token, 16 or 32 output rows): each rank's middle row
//              quantised, its down product, and the weighted sum in rank order
//              with the shared expert
// Both are bound by the experts' bytes (6 H I flops a token and expert against
// 3 H I bytes an expert): every byte of a reached expert's gate and up is read
// once however many tokens share it; down rows that tokens share are read by
// workgroups of one XCD at about the same time, so that its L2 serves them.
#include "moe_ffn.h"
#include "moe_fp8.hpp"

#include <algorithm>
#include <new>

namespace moe {

inline constexpr int kFp8LayerTokens = 64;   // tokens of one forward: one lane each in the grouping

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

inline constexpr int kChunk = 24;   // blocks of K whose rows a gate/up workgroup holds in LDS: 50 KB

// ------------------------------------------------------------ gate and up ---
// Workgroup (p, s): route p = t k + r (p = T k: the shared expert), rows 16 s
// .. + 15.  It goes on if no earlier route names the same expert and takes all
// tokens that do, in columns of 16.  Wave w multiplies blocks w, w + W, ..;
// the partial sums meet in LDS, in wave order.
template<int T_>
__global__ __launch_bounds__(512) void k_fp8_gate_up(Fp8LayerArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // x codes [blocks][2048], scales [blocks][16]; then the sums
    __shared__ int rank_of[kFp8LayerTokens], token[kFp8LayerTokens], rank[kFp8LayerTokens], counted;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    const int S = a.I / 16, s = blockIdx.x % S, p = blockIdx.x / S, routes = a.T * a.k;
    const bool shared = p == routes;
    if (s == 0 && !shared && p % a.k == 0) {
        // The token's input flags, whatever becomes of its routes.
        const size_t row = static_cast<size_t>(p / a.k) * a.H;
        bool bad = false;
        for (int i = threadIdx.x; i < a.H; i += blockDim.x) bad |= !isfinite(load1<T_>(a.x, row + i));
        if (bad) atomicOr(a.error, 1);
    }
    const int e = shared ? a.E : a.ids[p];
    if (!shared && (e < 0 || e >= a.E)) return;   // flagged by down_fold
    if (threadIdx.x < kFp8LayerTokens) rank_of[threadIdx.x] = shared && static_cast<int>(threadIdx.x) < a.T ? a.k : INT_MAX;
    __syncthreads();
    int earlier = 0;
    if (!shared) {
        for (int q = threadIdx.x; q < routes; q += blockDim.x) {
            if (a.ids[q] != e) continue;
            if (q < p) earlier = 1;
            atomicMin(&rank_of[q / a.k], q % a.k);
        }
    }
    if (__syncthreads_or(earlier)) return;
    if (wave == 0) {
        const int r = rank_of[lane];
        const uint64_t in = __builtin_amdgcn_ballot_w64(r != INT_MAX);
        if (r != INT_MAX) {
            const int at = __builtin_popcountll(in & ((uint64_t{1} << lane) - 1));
            token[at] = lane;
            rank[at] = r;
        }
        if (lane == 0) counted = __builtin_popcountll(in);
    }
    const size_t tile0 = (static_cast<size_t>(e) * S + s) * a.nbh;
    const uint8_t *gw = a.gate + tile0 * kFp8TileBytes, *uw = a.up + tile0 * kFp8TileBytes;
    const size_t scale0 = (static_cast<size_t>(e) * ((a.I + kFp8Block - 1) / kFp8Block) + s * 16 / kFp8Block) * a.nbh;
    const float *gs = a.gate_s + scale0, *us = a.up_s + scale0;
    constexpr int U = 2;   // blocks whose loads are in flight together
    __syncthreads();
    const int count = __builtin_amdgcn_readfirstlane(counted);

    for (int c0 = 0; c0 < count; c0 += 16) {
        const int cols = min(16, count - c0);
        f32x4 ga = {0.0f, 0.0f, 0.0f, 0.0f}, ua = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < a.nbh; k0 += kChunk) {
            const int kb = min(kChunk, a.nbh - k0);
            float *xs = reinterpret_cast<float *>(lds + kb * kFp8TileBytes);
            Frag gf[U], uf[U];
            auto load = [&](int b0) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    // Past the chunk: the round's first block again, not used below.
                    const int b = k0 + (b0 + u * W < kb ? b0 + u * W : b0);
                    gf[u] = load_tile(gw + static_cast<size_t>(b) * kFp8TileBytes, lane);
                    uf[u] = load_tile(uw + static_cast<size_t>(b) * kFp8TileBytes, lane);
                }
            };
            if (wave < kb) load(wave);
            // The columns' blocks, 16 threads each.
            for (int i = threadIdx.x >> 4; i < cols * kb; i += blockDim.x >> 4) {
                const int c = i / kb, b = i % kb, part = threadIdx.x & 15, col = (k0 + b) * kFp8Block + part * 8;
                Raw8 raw{};
                if (col < a.H) raw = load8_raw<T_>(a.x, static_cast<size_t>(token[c0 + c]) * a.H + col);
                float v[8];
                unpack8<T_>(raw, v);
                const GroupScale g = group_scale(max16(v));
                *reinterpret_cast<uint2 *>(lds + b * kFp8TileBytes + tile_offset(part, c)) = quantize8(v, g);
                if (part == 0) xs[b * 16 + c] = g.s;
            }
            __syncthreads();
            for (int b0 = wave; b0 < kb; b0 += W * U) {
                if (b0 != wave) load(b0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int b = b0 + u * W;
                    if (b >= kb) break;
                    const FragF16 x = to_f16(load_tile(lds + b * kFp8TileBytes, lane));
                    const float sx = xs[b * 16 + (lane & 15)];
                    const f32x4 gp = block_dot(to_f16(gf[u]), x), upr = block_dot(to_f16(uf[u]), x);
                    const float sg = sx * gs[k0 + b], su = sx * us[k0 + b];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        ga[q] = fmaf(gp[q], sg, ga[q]);
                        ua[q] = fmaf(upr[q], su, ua[q]);
                    }
                }
            }
            __syncthreads();   // the rows are used up
        }
        f32x4 *red = reinterpret_cast<f32x4 *>(lds);   // [wave][gate, up][lane]
        red[(wave * 2 + 0) * 64 + lane] = ga;
        red[(wave * 2 + 1) * 64 + lane] = ua;
        __syncthreads();
        // Sum i: row 4 (lane / 16) + i % 4 of column lane % 16, lane = i / 4.
        const float *sum = reinterpret_cast<const float *>(lds);
        int flags = 0;
        for (int i = threadIdx.x; i < 256; i += blockDim.x) {
            const int c = (i >> 2) & 15, row = (i >> 6) * 4 + (i & 3);
            if (c >= cols) continue;
            float g = sum[i], u = sum[256 + i];
            for (int q = 1; q < W; ++q) {
                g = g + sum[q * 512 + i];
                u = u + sum[q * 512 + 256 + i];
            }
            const size_t pair = static_cast<size_t>(token[c0 + c]) * a.P1 + rank[c0 + c];
            a.middle[pair * a.I + s * 16 + row] = silu_mul(g, u, flags);
        }
        if (flags) atomicOr(a.error, flags);
        __syncthreads();   // the sums are used up
    }
}

// ------------------------------------------------------- down and the sum ---
// Workgroup (t, slice of 16 RT rows); wave w takes ranks w, w + W, ..  All 16
// columns of its MFMA hold the one token, so every lane has its results.
template<int T_, int RT>
__global__ __launch_bounds__(1024) void k_fp8_down_fold(Fp8LayerArgs a) {
    constexpr int R = 16 * RT, MaxPairs = 33;
    constexpr int KB = 4;   // blocks in flight together: 64 lanes x 8 elements
    __shared__ __attribute__((aligned(16))) uint8_t codes[16][KB * kFp8Block];
    __shared__ float scales[16][KB];
    __shared__ float part[MaxPairs][R];
    __shared__ float weight[MaxPairs];
    __shared__ int valid[MaxPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    // Workgroup i runs on XCD i % 8: all tokens of one slice on one XCD, one
    // after the other, so that experts they share come from its L2.
    const int S = a.H / R, j = blockIdx.x >> 3, t = j % a.T, s = (blockIdx.x & 7) + 8 * (j / a.T);
    if (s >= S) return;
    const int m0 = s * R;
    int flags = 0;
    for (int r = wave; r < a.P1; r += W) {
        // The route: a bad id and a repeat of an earlier rank are dropped.
        int e = a.E;
        float w = 1.0f;
        if (r < a.k) {
            const int mine = lane < a.k ? a.ids[t * a.k + lane] : -1;
            w = a.weights[t * a.k + r];
            e = __builtin_amdgcn_readlane(mine, r);
            if (!isfinite(w) || w < 0.0f) flags |= 1;
            if (e < 0 || e >= a.E || __builtin_amdgcn_ballot_w64(lane < r && mine == e)) {
                flags |= 1;
                e = -1;
            }
        } else if (a.shared_gate) {
            w = a.shared_gate[t];
        }
        if (lane == 0) {
            weight[r] = w;
            valid[r] = e >= 0;
        }
        if (e < 0) continue;
        const uint8_t *dw = a.down + (static_cast<size_t>(e) * (a.H / 16) + m0 / 16) * a.nbi * kFp8TileBytes;
        const float *ds = a.down_s + (static_cast<size_t>(e) * ((a.H + kFp8Block - 1) / kFp8Block) + m0 / kFp8Block) * a.nbi;
        const float *mid = a.middle + (static_cast<size_t>(t) * a.P1 + r) * a.I;
        f32x4 acc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < a.nbi; k0 += KB) {
            const int kb = min(KB, a.nbi - k0);
            Frag wf[KB][RT];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int at = k0 + min(b, kb - 1);   // past the row's end: its last block again, not used
#pragma unroll
                for (int i = 0; i < RT; ++i) wf[b][i] = load_tile(dw + (static_cast<size_t>(i) * a.nbi + at) * kFp8TileBytes, lane);
            }
            // Lane l: elements 8 l .. + 7 of the row's next 512.
            const int col = k0 * kFp8Block + lane * 8;
            Raw8 raw{};
            if (col < a.I) raw = load8_raw<kF32>(mid, col);
            float v[8];
            unpack8<kF32>(raw, v);
            const GroupScale g = group_scale(max16(v));
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last round's reads are done
            *reinterpret_cast<uint2 *>(&codes[wave][lane * 8]) = quantize8(v, g);
            if ((lane & 15) == 0) scales[wave][lane >> 4] = g.s;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                if (b >= kb) break;
                const uint4 *c = reinterpret_cast<const uint4 *>(&codes[wave][b * kFp8Block + (lane >> 4) * 32]);
                const FragF16 x = to_f16(Frag{c[0], c[1]});
                const float sc = scales[wave][b] * ds[k0 + b];
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const f32x4 p = block_dot(to_f16(wf[b][i]), x);
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][q] = fmaf(p[q], sc, acc[i][q]);
                }
            }
        }
        if ((lane & 15) == 0) {
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) part[r][16 * i + (lane >> 4) * 4 + q] = acc[i][q];
        }
    }
    if (s == 0 && flags && lane == 0) atomicOr(a.error, flags);
    __syncthreads();
    if (threadIdx.x < R) {
        // y = +0 + w_0 c_0 + .. in rank order, + sigmoid(gate) shared, with the
        // flags of moe_ffn_forward's sum.
        const int row = threadIdx.x;
        int f = 0;
        float v = 0.0f;
        for (int r = 0; r < a.k; ++r) {
            if (!valid[r]) continue;
            float c = part[r][row], w = weight[r];
            if (!isfinite(c)) { f |= 1; c = 0.0f; }
            if (!isfinite(w)) { f |= 1; w = 0.0f; }
            float q = w * c;
            if (!isfinite(q)) { f |= 2; q = 0.0f; }
            v = v + q;
            if (!isfinite(v)) { f |= 2; v = 0.0f; }
        }
        if (f) v = 0.0f;
        int sf = 0;
        if (a.P1 > a.k) {
            float c = part[a.k][row], scale = 1.0f;
            if (!isfinite(c)) { sf |= 1; c = 0.0f; }
            if (a.shared_gate) {
                float g = weight[a.k];
                if (!isfinite(g)) { sf |= 1; g = 0.0f; }
                scale = 1.0f / (1.0f + moe_expf(-g));
                if (!isfinite(scale)) { sf |= 2; scale = 0.0f; }
            }
            const float q = scale * c;
            v = v + q;
            if (!isfinite(v)) { sf |= 2; v = 0.0f; }
        }
        store1<T_>(a.y, static_cast<size_t>(t) * a.H + m0 + row, sf ? 0.0f : v);
        if (f | sf) atomicOr(a.error, f | sf);
    }
}

template<int T_>
hipError_t launch_layer(const Fp8LayerArgs &a, hipStream_t s) {
    const int pairs = a.T * a.k + (a.P1 > a.k ? 1 : 0), W = std::min(8, a.nbh);
    const size_t rows = static_cast<size_t>(std::min(a.nbh, kChunk)) * (kFp8TileBytes + 64);
    const size_t lds = std::max<size_t>(rows, static_cast<size_t>(W) * 2048);
    k_fp8_gate_up<T_><<<dim3(static_cast<unsigned>(pairs) * (a.I / 16)), dim3(64 * W), lds, s>>>(a);
    hipError_t r = hipGetLastError();
    if (r != hipSuccess) return r;
    const int W2 = std::min(16, a.P1);
    const auto grid = [&](int rows_) { return dim3(static_cast<unsigned>((a.H / rows_ + 7) / 8 * 8) * a.T); };
    if (a.T >= 4) k_fp8_down_fold<T_, 2><<<grid(32), dim3(64 * W2), 0, s>>>(a);
    else k_fp8_down_fold<T_, 1><<<grid(16), dim3(64 * W2), 0, s>>>(a);
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
                                   p.cols, blocks(p.cols), nullptr);
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
    moe::LaunchDevice device(L->device);
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
