// Products of rows grouped by expert with a bank of int8 matrices (moe_i8_bank_*),
// and the routed-expert layer made of them (moe_i8_layer_*):
//   quantise x per token | group the routes by expert | gate and up, SiLU(g) u |
//   quantise each row of that | down | weighted sum in rank order with the shared
//   expert, which is the group behind the last
#include "moe_ffn.h"
#include "moe_i8.hpp"

#include <algorithm>
#include <new>

namespace moe {
namespace {

// The groups' row tiles, in LDS: first[e] = row tiles before group e, row[e] = its
// first row, both of E + 1 entries.  Offsets outside 0 .. N, or below the one
// before, are drawn into that range and set bit 1; a group ends where the next
// begins, and is empty where that is not after its own begin.
__device__ __forceinline__ int group_tiles(const I8Args &a, int BN, int *first, int *row) {
    __shared__ int sums[16];
    __shared__ int total;
    const int T = blockDim.x, per = (a.experts + T - 1) / T, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lo = min(a.experts, static_cast<int>(threadIdx.x) * per), hi = min(a.experts, lo + per);
    int bad = 0, mine = 0;
    for (int e = lo; e < hi; ++e) {
        const int from = a.offsets[e], to = a.offsets[e + 1], f = max(0, min(from, a.N)), t = max(0, min(to, a.N));
        if (f != from || t != to || t < f) bad = 1;
        row[e] = f;
        if (e + 1 == a.experts) row[e + 1] = t;
        first[e] = mine;
        mine += (max(t - f, 0) + BN - 1) / BN;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int before = incl - mine, all = 0;
    for (int w = 0; w < T / 64; ++w) {
        if (w < wave) before += sums[w];
        all += sums[w];
    }
    for (int e = lo; e < hi; ++e) first[e] += before;
    if (threadIdx.x == 0) {
        first[a.experts] = all;
        total = all;
    }
    if (bad && blockIdx.x == 0) atomicOr(a.error, 1);
    __syncthreads();
    return total;
}
// The last group e with first[e] <= t, which is the one that has row tile t: 64
// lanes look at every `step`-th entry and then at those between.
__device__ __forceinline__ int group_of(const int *first, int E, int t) {
    const int lane = threadIdx.x & 63, step = (E + 63) / 64;   // at most 64: E <= 4096
    int e = lane * step;
    const int s = __builtin_popcountll(__builtin_amdgcn_ballot_w64(e < E && first[min(e, E - 1)] <= t)) - 1;
    const int base = __builtin_amdgcn_readfirstlane(s) * step;
    e = base + lane;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < step && e < E && first[min(e, E - 1)] <= t)) - 1;
    return __builtin_amdgcn_readfirstlane(base + n);
}

// Workgroups take (row tile, matrix tile) items in turn; those of one XCD a run of
// their own, in which the matrix tiles of a row tile follow each other, so that an
// expert's matrix and its rows come from that XCD's L2 after the first time.
template<int WR, int WC, int TM, int TN, int S, int KS, int Form, int Y>
__global__ __launch_bounds__(64 * WR * WC) void k_i8_grouped(I8Args a) {
    using Tile = I8Tile<WR, WC, TM, TN, S, KS>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::Lds];
    extern __shared__ int table[];
    int *first = table, *row = table + a.experts + 1;
    const int items = group_tiles(a, Tile::BN, first, row) * a.tiles_m;
    const int each = (items + 7) / 8, end = min(items, static_cast<int>((blockIdx.x & 7) + 1) * each);
    int flags = 0;
    Tile g(lds);
    for (int i = static_cast<int>(blockIdx.x & 7) * each + static_cast<int>(blockIdx.x >> 3); i < end; i += gridDim.x >> 3) {
        const int t = i / a.tiles_m, m0 = i % a.tiles_m * Tile::BM;
        const int e = group_of(first, a.experts, t);
        const int r = __builtin_amdgcn_readfirstlane((t - first[e]) * Tile::BN + row[e]);
        const int cols = __builtin_amdgcn_readfirstlane(min(Tile::BN, row[e + 1] - r));
        g.start(a, e, m0, r, cols, flags);
        i32x4 acc[TM][TN];
        g.product(lds, acc);
        if constexpr (Form == kStoreMiddle) g.store_middle(a, e, m0, r, cols, acc, flags);
        else g.template store_rows<Y>(a, e, m0, r, cols, acc, lds);
        if constexpr (Form == kStoreRows && Y != kF32) __syncthreads();   // the results have left the buffers
    }
    if (flags) atomicOr(a.error, flags);
}

template<int WR, int WC, int TM, int TN, int S, int KS, int Form, int Y>
hipError_t launch_tile(I8Args a, hipStream_t s) {
    using Tile = I8Tile<WR, WC, TM, TN, S, KS>;
    a.tiles_m = (a.M + Tile::BM - 1) / Tile::BM;
    const size_t lds = static_cast<size_t>(a.experts + 1) * 8;
    const int resident = std::max(1, static_cast<int>(160 * 1024 / (Tile::Lds + lds + 256)));
    const size_t items = (static_cast<size_t>(a.N) / Tile::BN + std::min(a.N, a.experts)) * a.tiles_m;   // at most
    const size_t grid = std::min((items + 7) / 8 * 8, static_cast<size_t>(256) * std::min(resident, 4));
    k_i8_grouped<WR, WC, TM, TN, S, KS, Form, Y><<<dim3(static_cast<unsigned>(grid)), dim3(64 * Tile::W), lds, s>>>(a);
    return hipGetLastError();
}

template<int Form, int Y>
hipError_t launch_grouped(const I8Args &a, hipStream_t s) {
    const int mean = a.N / a.experts;
    if (mean <= 12) return launch_tile<4, 1, 2, 1, 3, 4, Form, Y>(a, s);
    if (mean <= 64) return launch_tile<2, 2, 2, 2, 3, 2, Form, Y>(a, s);
    return launch_tile<2, 2, 4, 4, 4, 1, Form, Y>(a, s);
}

hipError_t launch_grouped_rows(const I8Args &a, int y_type, hipStream_t s) {
    if (y_type == kF32) return launch_grouped<kStoreRows, kF32>(a, s);
    if (y_type == kBF16) return launch_grouped<kStoreRows, kBF16>(a, s);
    return launch_grouped<kStoreRows, kF16>(a, s);
}

// y = +0 + w_0 c_0 + .. in rank order, + sigmoid(gate) shared, with the flags of
// moe_ffn_forward's sum, rounded once; four elements a thread.  c: grouped rows.
struct I8FoldArgs {
    const float *c;            // [pairs][H]
    const int32_t *pos_of;     // [tokens * k] row of c, -1 for a route that was dropped
    const int32_t *offsets;    // [E + 2]; the shared expert's rows begin at offsets[E]
    const float *weights, *shared_gate;
    void *y;
    int tokens, H, k, E, shared;
    int *error;
};
template<int T>
__global__ __launch_bounds__(256) void k_i8_fold(I8FoldArgs a) {
    const size_t i = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (i >= static_cast<size_t>(a.tokens) * a.H) return;
    const size_t t = i / a.H, h = i % a.H;
    typedef float f4 __attribute__((ext_vector_type(4)));
    const auto load = [&](size_t row) { return __builtin_nontemporal_load(reinterpret_cast<const f4 *>(a.c + row * a.H + h)); };
    int flags[4] = {};
    float v[4] = {};
    for (int r0 = 0; r0 < a.k; r0 += 8) {
        f4 x[8];
        float w[8];
        int pos[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            pos[q] = r0 + q < a.k ? a.pos_of[t * a.k + r0 + q] : -1;
            if (pos[q] >= 0) x[q] = load(pos[q]);
            w[q] = r0 + q < a.k ? a.weights[t * a.k + r0 + q] : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (pos[q] < 0) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float c = x[q][e], s = w[q];
                if (!isfinite(c)) { flags[e] |= 1; c = 0.0f; }
                if (!isfinite(s)) { flags[e] |= 1; s = 0.0f; }
                float p = s * c;
                if (!isfinite(p)) { flags[e] |= 2; p = 0.0f; }
                v[e] = v[e] + p;
                if (!isfinite(v[e])) { flags[e] |= 2; v[e] = 0.0f; }
            }
        }
    }
    int any = 0;
    f4 sx = {0.0f, 0.0f, 0.0f, 0.0f};
    float scale = 1.0f;
    int gate_flags = 0;
    if (a.shared) {
        sx = load(a.offsets[a.E] + t);
        if (a.shared_gate) {
            float g = a.shared_gate[t];
            if (!isfinite(g)) { gate_flags |= 1; g = 0.0f; }
            scale = 1.0f / (1.0f + moe_expf(-g));
            if (!isfinite(scale)) { gate_flags |= 2; scale = 0.0f; }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (flags[e]) v[e] = 0.0f;
        int sf = 0;
        if (a.shared) {
            sf = gate_flags;
            float c = sx[e];
            if (!isfinite(c)) { sf |= 1; c = 0.0f; }
            v[e] = v[e] + scale * c;
            if (!isfinite(v[e])) { sf |= 2; v[e] = 0.0f; }
            if (sf) v[e] = 0.0f;
        }
        any |= flags[e] | sf;
    }
    store4<T>(a.y, i, v);
    if (any) atomicOr(a.error, any);
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_i8_bank {
    int experts = 0, input = 0, output = 0, device = 0;
    uint8_t *mem = nullptr;   // tiles, scales
    const float *scales = nullptr;
};

struct moe_i8_layer {
    moe_i8_layer_config cfg{};
    int device = 0;
    uint8_t *mem = nullptr;                        // weights
    const uint8_t *gate_up = nullptr, *down = nullptr;
    const float *gate_up_s = nullptr, *down_s = nullptr;
    uint8_t *ws = nullptr;
    int64_t x_pitch = 0, m_pitch = 0;
    int8_t *x = nullptr, *m = nullptr;             // quantised rows of x and of the middle
    float *x_s = nullptr, *m_s = nullptr;
    float *middle = nullptr, *contrib = nullptr;   // [pairs][I], [pairs][H]
    int *dropped = nullptr;                        // flags of rows that are not used
    moe::RouteOut routes{};
};

namespace {

constexpr int kInvalid = hipErrorInvalidValue;

bool aligned(const void *p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }
bool is_type(int t) { return t == MOE_F32 || t == MOE_BF16 || t == MOE_F16; }
int64_t odd_pitch(int width) { return static_cast<int64_t>(moe::i8_chunks(width) | 1) * moe::kI8Chunk; }
size_t tile_bytes(int rows, int cols) { return static_cast<size_t>((rows + 15) / 16) * moe::i8_chunks(cols) * moe::kI8TileBytes; }

// `count` matrices of codes on the host or the device into tiles at `to`.
hipError_t upload(const void *codes, uint8_t *to, size_t count, int rows, int cols, bool pairs, int shift, bool on_device) {
    if (on_device) return moe::launch_i8_repack(static_cast<const int8_t *>(codes), to, count, rows, cols, pairs, shift, nullptr);
    void *staging = nullptr;
    const size_t bytes = count * rows * cols;
    hipError_t r = hipMalloc(&staging, bytes);
    if (r == hipSuccess) r = hipMemcpy(staging, codes, bytes, hipMemcpyHostToDevice);
    if (r == hipSuccess) r = moe::launch_i8_repack(static_cast<const int8_t *>(staging), to, count, rows, cols, pairs, shift, nullptr);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (staging) (void)hipFree(staging);
    return r;
}

bool valid_config(const moe_i8_layer_config *c) {
    return c && c->hidden >= 32 && c->hidden <= 16384 && c->hidden % 32 == 0 && c->intermediate >= 32 &&
           c->intermediate <= 16384 && c->intermediate % 32 == 0 && c->experts >= 1 && c->experts <= 4096 - c->has_shared && c->top_k >= 1 &&
           c->top_k <= 32 && c->top_k <= c->experts && (c->has_shared == 0 || c->has_shared == 1) && c->max_tokens >= 1 &&
           c->max_tokens <= 65536;
}

struct LayerLayout {
    size_t gate_up, down, gate_up_s, down_s, weights;   // offsets and end of the weights
    size_t x, x_s, m, m_s, middle, contrib, counts, offsets, token, rank, pos, stream_items, mfma_items, item_counts, dropped, bitmap,
        prefix, workspace;
};
LayerLayout layout(const moe_i8_layer_config &c) {
    LayerLayout l{};
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    const size_t H = c.hidden, I = c.intermediate, Ep = static_cast<size_t>(c.experts) + c.has_shared, T = c.max_tokens;
    const size_t P = T * (c.top_k + c.has_shared), W = (T + 31) / 32;
    l.gate_up = take(Ep * 2 * tile_bytes(c.intermediate, c.hidden));
    l.down = take(Ep * tile_bytes(c.hidden, c.intermediate));
    l.gate_up_s = take(Ep * 2 * I * 4);
    l.down_s = take(Ep * H * 4);
    l.weights = at;
    at = 0;
    l.x = take(T * odd_pitch(c.hidden));
    l.x_s = take(T * 4);
    l.m = take(P * odd_pitch(c.intermediate));
    l.m_s = take(P * 4);
    l.middle = take(P * I * 4);
    l.contrib = take(P * H * 4);
    l.counts = take(Ep * 4);
    l.offsets = take((Ep + 1) * 4);
    l.token = take(P * 4);
    l.rank = take(P * 4);
    l.pos = take(T * c.top_k * 4);
    l.stream_items = take(sizeof(moe::Item));
    l.mfma_items = take((P / moe::kMfmaTile + std::min(P, Ep)) * sizeof(moe::Item));
    l.item_counts = take(16);
    l.dropped = take(4);
    l.bitmap = take(W * Ep * 4);
    l.prefix = take(W * Ep * 4);
    l.workspace = at;
    return l;
}

void release(moe_i8_bank *B) {
    if (B->mem) (void)hipFree(B->mem);
    delete B;
}
void release(moe_i8_layer *L) {
    if (L->mem) (void)hipFree(L->mem);
    if (L->ws) (void)hipFree(L->ws);
    delete L;
}

}  // namespace

extern "C" {

int moe_i8_bank_create(int experts, int input, int output, const void *codes, const float *scales, int weights_on_device,
                       int device, moe_i8_bank **out) {
    if (!out) return kInvalid;
    *out = nullptr;
    if (experts < 1 || experts > 4096 || input < 32 || input > 16384 || input % 32 || output < 1 || output > 65536 || !codes ||
        !aligned(scales, 4) || device < 0)
        return kInvalid;
    moe::DeviceScope scope(device);
    if (!scope.ok()) return hipErrorInvalidDevice;
    auto *B = new (std::nothrow) moe_i8_bank;
    if (!B) return hipErrorOutOfMemory;
    B->experts = experts;
    B->input = input;
    B->output = output;
    B->device = device;
    const size_t scale_at = round_up(tile_bytes(output, input) * experts, 256), scale_bytes = static_cast<size_t>(experts) * output * 4;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&B->mem, scale_at + scale_bytes);
    if (r == hipSuccess) r = upload(codes, B->mem, experts, output, input, false, 0, weights_on_device != 0);
    if (r == hipSuccess)
        r = hipMemcpy(B->mem + scale_at, scales, scale_bytes, weights_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (r != hipSuccess) { release(B); return r; }
    B->scales = reinterpret_cast<const float *>(B->mem + scale_at);
    *out = B;
    return 0;
}

int moe_i8_bank_destroy(moe_i8_bank *B) {
    if (!B) return kInvalid;
    moe::DeviceScope scope(B->device);
    release(B);
    return 0;
}

int moe_i8_bank_bytes(const moe_i8_bank *B, size_t *weight_bytes) {
    if (!B || !weight_bytes) return kInvalid;
    *weight_bytes = static_cast<size_t>(B->experts) * B->output * (static_cast<size_t>(B->input) + 4);
    return 0;
}

int moe_i8_bank_forward(moe_i8_bank *B, const void *x_codes, const float *x_scales, int x_rows, const int32_t *index,
                        const int32_t *offsets, int rows, void *y, int y_type, int64_t y_stride, int *error, void *stream) {
    if (!B || !aligned(x_codes, 16) || !aligned(x_scales, 4) || x_rows < 1 || x_rows > (1 << 22) || rows < 1 ||
        rows > (1 << 22) || (index && !aligned(index, 4)) || !aligned(offsets, 4) || !is_type(y_type) ||
        !aligned(y, moe::elem_bytes(y_type)) || y_stride < B->output || y_stride > (int64_t{1} << 40) || !aligned(error, 4))
        return kInvalid;
    // Without an index the rows are those of x; with one they are reached by 32-bit offsets.
    if (index ? static_cast<int64_t>(x_rows) * B->input > (int64_t{1} << 31) : rows > x_rows) return kInvalid;
    moe::DeviceScope device(B->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    moe::I8Args a{};
    a.tiles = B->mem;
    a.sw = B->scales;
    a.x = static_cast<const int8_t *>(x_codes);
    a.sx = x_scales;
    a.pitch = B->input;
    a.index = index;
    a.x_rows = x_rows;
    a.offsets = offsets;
    a.experts = B->experts;
    a.y = y;
    a.y_stride = y_stride;
    a.M = B->output;
    a.N = rows;
    a.K = B->input;
    a.chunks = moe::i8_chunks(B->input);
    a.error = error;
    return moe::launch_grouped_rows(a, y_type, static_cast<hipStream_t>(stream));
}

int moe_i8_layer_memory_bytes(const moe_i8_layer_config *c, size_t *weight_bytes, size_t *workspace_bytes) {
    if (!valid_config(c) || !weight_bytes || !workspace_bytes) return kInvalid;
    const LayerLayout l = layout(*c);
    *weight_bytes = l.weights;
    *workspace_bytes = l.workspace;
    return 0;
}

int moe_i8_layer_create(const moe_i8_layer_config *c, const moe_i8_matrix *experts, const moe_i8_matrix *shared,
                        int weights_on_device, int device, moe_i8_layer **out) {
    if (!out) return kInvalid;
    *out = nullptr;
    if (!valid_config(c) || !experts || (c->has_shared && !shared) || device < 0) return kInvalid;
    for (int i = 0; i < 3; ++i) {
        if (!experts[i].codes || !aligned(experts[i].scales, 4)) return kInvalid;
        if (c->has_shared && (!shared[i].codes || !aligned(shared[i].scales, 4))) return kInvalid;
    }
    moe::DeviceScope scope(device);
    if (!scope.ok()) return hipErrorInvalidDevice;
    auto *L = new (std::nothrow) moe_i8_layer;
    if (!L) return hipErrorOutOfMemory;
    L->cfg = *c;
    L->device = device;
    L->x_pitch = odd_pitch(c->hidden);
    L->m_pitch = odd_pitch(c->intermediate);
    const LayerLayout l = layout(*c);
    const bool on_device = weights_on_device != 0;
    const int H = c->hidden, I = c->intermediate;
    const size_t E = c->experts, one = tile_bytes(I, H), half = static_cast<size_t>(I) * 4;
    const hipMemcpyKind kind = on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, l.weights);
    if (r == hipSuccess) r = hipMalloc(&L->ws, l.workspace);
    const auto bank = [&](const moe_i8_matrix *m, size_t at, size_t count) {
        for (int i = 0; i < 2 && r == hipSuccess; ++i) {
            r = upload(m[i].codes, L->mem + l.gate_up + at * 2 * one, count, I, H, true, i, on_device);
            // Scales in the order of the rows: 16 of gate, 16 of up.
            if (r == hipSuccess)
                r = hipMemcpy2D(L->mem + l.gate_up_s + at * 2 * half + i * 64, 128, m[i].scales, 64, 64, count * (I / 16), kind);
        }
        if (r == hipSuccess) r = upload(m[2].codes, L->mem + l.down + at * tile_bytes(H, I), count, H, I, false, 0, on_device);
        if (r == hipSuccess) r = hipMemcpy(L->mem + l.down_s + at * H * 4, m[2].scales, count * H * 4, kind);
    };
    if (r == hipSuccess) bank(experts, 0, E);
    if (r == hipSuccess && c->has_shared) bank(shared, E, 1);
    if (r == hipSuccess) r = hipDeviceSynchronize();
    if (r != hipSuccess) { release(L); return r; }
    L->gate_up = L->mem + l.gate_up;
    L->down = L->mem + l.down;
    L->gate_up_s = reinterpret_cast<const float *>(L->mem + l.gate_up_s);
    L->down_s = reinterpret_cast<const float *>(L->mem + l.down_s);
    L->x = reinterpret_cast<int8_t *>(L->ws + l.x);
    L->m = reinterpret_cast<int8_t *>(L->ws + l.m);
    L->x_s = reinterpret_cast<float *>(L->ws + l.x_s);
    L->m_s = reinterpret_cast<float *>(L->ws + l.m_s);
    L->middle = reinterpret_cast<float *>(L->ws + l.middle);
    L->contrib = reinterpret_cast<float *>(L->ws + l.contrib);
    const auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(L->ws + at); };
    L->dropped = ints(l.dropped);
    L->routes.counts = ints(l.counts);
    L->routes.offsets = ints(l.offsets);
    L->routes.pair_token = ints(l.token);
    L->routes.pair_rank = ints(l.rank);
    L->routes.pos_of = ints(l.pos);
    L->routes.stream_items = reinterpret_cast<moe::Item *>(L->ws + l.stream_items);
    L->routes.mfma_items = reinterpret_cast<moe::Item *>(L->ws + l.mfma_items);
    L->routes.item_counts = ints(l.item_counts);
    L->routes.bitmap = reinterpret_cast<uint32_t *>(L->ws + l.bitmap);
    L->routes.wprefix = reinterpret_cast<uint32_t *>(L->ws + l.prefix);
    *out = L;
    return 0;
}

int moe_i8_layer_destroy(moe_i8_layer *L) {
    if (!L) return kInvalid;
    moe::DeviceScope scope(L->device);
    release(L);
    return 0;
}

int moe_i8_layer_forward(moe_i8_layer *L, const void *x, int type, const int32_t *ids, const float *weights, int tokens,
                         const float *shared_gate, void *y, int *error, void *stream) {
    if (!L || !is_type(type) || tokens < 1 || tokens > L->cfg.max_tokens || !aligned(x, moe::elem_bytes(type)) ||
        !aligned(ids, 4) || !aligned(weights, 4) || (shared_gate && !aligned(shared_gate, 4)) ||
        !aligned(y, moe::elem_bytes(type)) || !aligned(error, 4))
        return kInvalid;
    moe::DeviceScope device(L->device);
    if (!device.ok()) return hipErrorInvalidDevice;
    const auto s = static_cast<hipStream_t>(stream);
    const moe_i8_layer_config &c = L->cfg;
    const int Ep = c.experts + c.has_shared, pairs = tokens * (c.top_k + c.has_shared);
    hipError_t r = moe::launch_quantize_i8(x, type, c.hidden, c.hidden, tokens, L->x, L->x_pitch, L->x_s, error, s);
    if (r != hipSuccess) return r;
    const moe::Shape shape{c.hidden, c.intermediate, c.experts, Ep, c.top_k};
    // Every group an item of the matrix kernels, of which only counts and positions are read.
    r = moe::launch_prepare(nullptr, ids, weights, tokens, shape, moe::ActOut{}, L->routes, 1, error, s);
    if (r != hipSuccess) return r;
    moe::I8Args a{};
    a.tiles = L->gate_up;
    a.sw = L->gate_up_s;
    a.x = L->x;
    a.sx = L->x_s;
    a.pitch = L->x_pitch;
    a.index = L->routes.pair_token;
    a.x_rows = tokens;
    a.offsets = L->routes.offsets;
    a.experts = Ep;
    a.y = L->middle;
    a.y_stride = c.intermediate;
    a.M = 2 * c.intermediate;
    a.N = pairs;
    a.K = c.hidden;
    a.chunks = moe::i8_chunks(c.hidden);
    a.error = error;
    if ((r = moe::launch_grouped<moe::kStoreMiddle, moe::kF32>(a, s)) != hipSuccess) return r;
    // Rows that no group took (dropped routes) are quantised as well, and not used;
    // what they hold raises no flag of this call, and SiLU(g) u is always finite.
    r = moe::launch_quantize_i8(L->middle, moe::kF32, c.intermediate, c.intermediate, pairs, L->m, L->m_pitch, L->m_s,
                                L->dropped, s);
    if (r != hipSuccess) return r;
    a.tiles = L->down;
    a.sw = L->down_s;
    a.x = L->m;
    a.sx = L->m_s;
    a.pitch = L->m_pitch;
    a.index = nullptr;
    a.x_rows = pairs;
    a.y = L->contrib;
    a.y_stride = c.hidden;
    a.M = c.hidden;
    a.K = c.intermediate;
    a.chunks = moe::i8_chunks(c.intermediate);
    if ((r = moe::launch_grouped<moe::kStoreRows, moe::kF32>(a, s)) != hipSuccess) return r;
    const moe::I8FoldArgs f{L->contrib, L->routes.pos_of, L->routes.offsets, weights, shared_gate, y,
                            tokens,     c.hidden,         c.top_k,           c.experts, c.has_shared, error};
    const dim3 grid(static_cast<unsigned>((static_cast<size_t>(tokens) * c.hidden / 4 + 255) / 256)), block(256);
    if (type == MOE_F32) moe::k_i8_fold<moe::kF32><<<grid, block, 0, s>>>(f);
    else if (type == MOE_BF16) moe::k_i8_fold<moe::kBF16><<<grid, block, 0, s>>>(f);
    else moe::k_i8_fold<moe::kF16><<<grid, block, 0, s>>>(f);
    return hipGetLastError();
}

}  // extern "C"
