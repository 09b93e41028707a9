// Products of rows grouped by expert with a bank of int8 matrices (moe_i8_bank_*),
// and the routed-expert layer made of them (moe_i8_layer_*):
//   quantise x per token | group the routes by expert | gate and up, SiLU(g) u |
//   quantise each row of that | down | weighted sum in rank order with the shared
//   expert, which is the group behind the last
#include "moe_ffn.h"
#include "moe_i8.hpp"

#include <algorithm>
#include <cmath>
#include <new>

namespace moe {
namespace {

// The groups' row tiles, in LDS: group list[p] has the row tiles from first[p] to
// first[p + 1], and its rows begin at row[e].  Groups of more than one tile come
// first, with `big` tiles between them.  Offsets outside 0 .. N are drawn into that
// range, those below one before up to it, so that no row has two groups and the
// tiles are at most N / BN and one a group; they set bit 1.
inline constexpr int kMostExperts = 4096;
struct GroupTable {
    int *first, *list, *row;   // [E + 1], [E], [E + 1]
    int experts, tiles, big;

    static constexpr size_t bytes(int experts) { return (static_cast<size_t>(experts) * 3 + 2) * 4; }
    static constexpr size_t kShared = 16 * 5 * 4;   // and of its own

    __device__ __forceinline__ GroupTable(const I8Args &a, int BN, int *lds) : experts(a.experts) {
        __shared__ int sums[16][4], wrong[16];
        first = lds;
        row = first + experts + 1;
        list = row + experts + 1;
        const int T = blockDim.x, per = (experts + T - 1) / T, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int lo = min(experts, static_cast<int>(threadIdx.x) * per), hi = min(experts, lo + per);
        bool bad = false;
        for (int e = lo; e < hi; ++e) {
            const int from = a.offsets[e], to = a.offsets[e + 1];
            bad |= from < 0 || to < from || to > a.N;
            row[e] = max(0, min(from, a.N));
            if (e + 1 == experts) row[e + 1] = max(0, min(to, a.N));
        }
        const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
        if (lane == 0) wrong[wave] = any != 0;
        __syncthreads();
        bad = false;
        for (int w = 0; w < T / 64; ++w) bad |= wrong[w] != 0;
        if (bad) {
            if (threadIdx.x == 0) {
                for (int e = 0; e < experts; ++e) row[e + 1] = max(row[e + 1], row[e]);
                if (blockIdx.x == 0) atomicOr(a.error, 1);
            }
            __syncthreads();
        }
        int mine[4] = {};   // big groups, their tiles, other groups, their tiles
        for (int e = lo; e < hi; ++e) {
            const int n = (row[e + 1] - row[e] + BN - 1) / BN, c = n > 1 ? 0 : 2;
            mine[c] += 1;
            mine[c + 1] += n;
        }
        int incl[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            incl[c] = mine[c];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(incl[c], d, 64);
                if (lane >= d) incl[c] += v;
            }
            if (lane == 63) sums[wave][c] = incl[c];
        }
        __syncthreads();
        int all[4] = {};
        for (int w = 0; w < T / 64; ++w) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (w < wave) incl[c] += sums[w][c];
                all[c] += sums[w][c];
            }
        }
        int at[2] = {incl[0] - mine[0], all[0] + incl[2] - mine[2]}, tile[2] = {incl[1] - mine[1], all[1] + incl[3] - mine[3]};
        for (int e = lo; e < hi; ++e) {
            const int n = (row[e + 1] - row[e] + BN - 1) / BN, c = n > 1 ? 0 : 1;
            list[at[c]] = e;
            first[at[c]] = tile[c];
            ++at[c];
            tile[c] += n;
        }
        tiles = __builtin_amdgcn_readfirstlane(all[1] + all[3]);
        big = __builtin_amdgcn_readfirstlane(all[1]);
        if (threadIdx.x == 0) first[experts] = tiles;
        __syncthreads();
    }
    // The last place p with first[p] <= t, whose group has row tile t: 64 lanes look
    // at every `step`-th place and then at those between.
    __device__ __forceinline__ int place(int t) const {
        const int lane = threadIdx.x & 63, step = (experts + 63) / 64;   // at most 64
        const auto before = [&](int p, bool in) { return in && p < experts && first[min(p, experts - 1)] <= t; };
        const int base = (__builtin_popcountll(__builtin_amdgcn_ballot_w64(before(lane * step, true))) - 1) * step;
        return base + __builtin_popcountll(__builtin_amdgcn_ballot_w64(before(base + lane, lane < step))) - 1;
    }
    __device__ __forceinline__ I8Item item(int t, int m0, int BN) const {
        const int p = __builtin_amdgcn_readfirstlane(place(t)), e = __builtin_amdgcn_readfirstlane(list[p]);
        const int r = __builtin_amdgcn_readfirstlane(row[e] + (t - first[p]) * BN);
        return I8Item{e, m0, r, __builtin_amdgcn_readfirstlane(min(BN, row[e + 1] - r)), t >= big};
    }
};

// Workgroups take (row tile, matrix tile) items in turn; those of one XCD a share
// of their own, in which the matrix tiles of a row tile follow each other, so that
// an expert's matrix and its rows come from that XCD's L2 after the first time.
// Where there are both, half of an XCD's workgroups begin with the groups of many
// tiles, whose products keep the matrix cores busy, and the other half with those
// whose matrices are read for a few rows; each has as many of either.
template<int WR, int WC, int TM, int TN, int S, int KS, int Form, int Y>
__global__ __launch_bounds__(64 * WR * WC) void k_i8_grouped(I8Args a) {
    using Stream = I8Stream<WR, WC, TM, TN, S, KS, Form, Y, true>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Stream::Lds];
    extern __shared__ int table[];
    const GroupTable groups(a, Stream::BN, table);
    const int xcd = static_cast<int>(blockIdx.x & 7), q = static_cast<int>(blockIdx.x >> 3), W = static_cast<int>(gridDim.x >> 3);
    // The XCD's share of the items of either kind: `big` and `rest` of them.
    const auto part = [](int n, int x) { return static_cast<int>(static_cast<int64_t>(n) * x / 8); };
    const int bigs = groups.big * a.tiles_m, rests = groups.tiles * a.tiles_m - bigs;
    int big0 = part(bigs, xcd), big = part(bigs, xcd + 1) - big0;
    int rest0 = bigs + part(rests, xcd), rest = bigs + part(rests, xcd + 1) - rest0;
    // Every other workgroup takes the second half of both kinds, the rest first.
    int from = q, step = W;
    bool rest_first = false;
    if (W > 1 && 8 * big >= rest && 8 * rest >= big) {
        const int half = q & 1;
        rest_first = half;
        from = q >> 1;
        step = (W + 1 - half) / 2;
        big0 += half * (big / 2);
        big = half ? big - big / 2 : big / 2;
        rest0 += half * (rest / 2);
        rest = half ? rest - rest / 2 : rest / 2;
    }
    const auto fetch = [&](int i) {
        const int j = rest_first ? (i < rest ? rest0 + i : big0 + i - rest) : (i < big ? big0 + i : rest0 + i - big);
        return groups.item(j / a.tiles_m, j % a.tiles_m * Stream::BM, Stream::BN);
    };
    Stream g(a, lds);
    g.run(from, step, big + rest, fetch,
          [&](const I8Item &it, const float *params, const i32x4 (&acc)[TM][TN]) {
              if constexpr (Form == kStoreMiddle) g.store_middle(it, params, acc);
              else g.store_rows(it, params, acc);
          });
    if (g.flags) atomicOr(a.error, g.flags);
}

template<int WR, int WC, int TM, int TN, int S, int KS, int Form, int Y>
hipError_t launch_tile(I8Args a, hipStream_t s) {
    using Stream = I8Stream<WR, WC, TM, TN, S, KS, Form, Y, true>;
    static_assert(Stream::Lds + GroupTable::bytes(kMostExperts) + GroupTable::kShared <= 160 * 1024, "a CU's LDS");
    a.tiles_m = (a.rows + Stream::BM - 1) / Stream::BM;
    const size_t lds = GroupTable::bytes(a.experts);
    const int resident = std::max(1, static_cast<int>(160 * 1024 / (Stream::Lds + lds + GroupTable::kShared)));
    const size_t items = (static_cast<size_t>(a.N) / Stream::BN + std::min(a.N, a.experts)) * a.tiles_m;   // at most
    const size_t grid = std::min((items + 7) / 8 * 8, static_cast<size_t>(256) * std::min(resident, 8));
    k_i8_grouped<WR, WC, TM, TN, S, KS, Form, Y><<<dim3(static_cast<unsigned>(grid)), dim3(64 * Stream::W), lds, s>>>(a);
    return hipGetLastError();
}

// The tile by the mean number of rows of a group, which the host knows: few rows,
// matrices read for them and workgroups enough to have many on their way; many
// rows, tiles that read less.  us, bank of 512 2048 x 1024 matrices, bf16, at 10, 80,
// 640, 2,560, 5,120 and 20,480 rows in even groups, then 10,320 of 2560 x 640 in uneven
// ones, fp32:
//   64 x 16     9.8 / 30.6 / 119 / 166 / 181 / 398 / 210
//   64 x 32    11.8 / 31.3 / 114 / 164 / 176 / 276 / 162
//   128 x 64   16.1 / 36.3 / 119 / 167 / 176 / 215 / 155
//   256 x 128  21.0 / 42.0 / 125 / 172 / 183 / 209 / 179
// The layer's gate and up, 64 x 32 / 128 x 32 / 128 x 64 / 256 x 128, all of the
// layer: 128 tokens - / 258 / 262 / 275, 512 - / 313 / 316 / 327, 1,024 - / 353 / 347 / 361,
// 4,096 - / 679 / 562 / 529; its down (K = 512, an item's start and end weigh more), 64 x 32 /
// 128 x 64 / 256 x 128: 128 tokens 274 / 265 / 274, 512 335 / 321 / 329, 4,096 671 / 614 / 530.
// A few experts: smaller tiles where larger ones leave CUs without any.  Bank of 8
// such matrices at 100, 300, 1,000 and 4,000 rows, bf16:
//   64 x 16                          7.7 / 10.7 / 24.1 / 64.2
//   64 x 32, stages of four chunks   8.0 / 10.4 / 18.9 / 42.3
//   64 x 32                          8.6 / 11.8 / 19.5 / 38.6
//   128 x 64                        10.9 / 15.2 / 13.7 / 24.8
//   256 x 128                       15.6 / 21.5 / 25.6 / 23.9
// Layer of 8 experts, 2048/512, top-2, gate and up by 64 x 32 / 128 x 32 / 128 x 64 / 256 x 128:
// 33 tokens 28.6 / 31.0 / 33.9 / 39.4, 400 37.0 / 34.4 / 38.5 / 47.9, 1,000 59.1 / 56.6 / 48.6 / 54.4.
template<int Form, int Y>
hipError_t launch_grouped(const I8Args &a, hipStream_t s) {
    const int mean = a.N / a.experts;
    // Tiles of groups that end, on average, in the middle of one.
    const auto tiles = [&](int m, int n) { return static_cast<int64_t>((a.rows + m - 1) / m) * (a.N / n + (std::min(a.N, a.experts) + 1) / 2); };
    if (mean > 64 && tiles(256, 128) >= 128) return launch_tile<4, 2, 4, 4, 4, 1, Form, Y>(a, s);
    if constexpr (Form == kStoreMiddle) {   // pairs of tiles
        if (tiles(64, 32) <= 256) return launch_tile<2, 2, 2, 1, 4, 4, Form, Y>(a, s);
        if (mean <= 12 || tiles(128, 64) <= 256) return launch_tile<4, 1, 2, 2, 4, 2, Form, Y>(a, s);
    } else {
        if (a.N <= a.experts / 2 || tiles(64, 16) <= 256) return launch_tile<4, 1, 1, 1, 4, 4, Form, Y>(a, s);
        if (tiles(64, 32) <= 256) return launch_tile<2, 2, 2, 1, 4, 4, Form, Y>(a, s);
        if (mean <= 12 && a.chunks > 16) return launch_tile<4, 1, 1, 2, 4, 2, Form, Y>(a, s);
    }
    return launch_tile<4, 1, 2, 4, 4, 1, Form, Y>(a, s);
}

hipError_t launch_grouped_rows(const I8Args &a, int y_type, hipStream_t s) {
    if (y_type == kF32) return launch_grouped<kStoreRows, kF32>(a, s);
    if (y_type == kBF16) return launch_grouped<kStoreRows, kBF16>(a, s);
    return launch_grouped<kStoreRows, kF16>(a, s);
}

// ------------------------------------------------------------- grouping ---
// Rows of the product ("pairs" of a token and one of its ranks) grouped by expert,
// the shared expert's behind the last.  Their order within a group is that in
// which LDS counted them, which nothing depends on: a row's result is the same
// wherever it stands, and the sum finds it by its place.
struct I8Groups {
    int32_t *offsets;   // [E' + 1]
    int32_t *token;     // [pairs]: token of a place
    int32_t *place;     // [tokens * k]: place of a route; -1: dropped
    int32_t *counts;    // [blocks][E']: routes of a block of tokens, for batches of many
    int4 *active;       // few tokens: expert, first place and number of rows of each group that has any
    int32_t *groups;    // and how many those are
};
struct I8GroupArgs {
    const int32_t *ids;
    const float *weights;
    I8Groups g;
    int tokens, k, E, Ep;
    int per, blocks;    // tokens of a block, blocks
    int *error;
};
inline constexpr int kGroupThreads = 256;

// The routes of tokens t0 .. t0 + n - 1, as they stand in sid (LDS): each one's
// number among the block's of its expert, or -1 for a bad id or an id of an earlier
// rank, to local(i, number); counts (LDS, zeroed) get the experts' numbers.
template<class Local>
__device__ __forceinline__ void count_routes(const I8GroupArgs &a, int t0, int n, int32_t *sid, int32_t *counts, const Local &local) {
    const size_t at = static_cast<size_t>(t0) * a.k;
    int flags = 0;
    for (int e = threadIdx.x; e < a.Ep; e += kGroupThreads) counts[e] = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n * a.k; i += kGroupThreads) {
        sid[i] = a.ids[at + i];
        const float w = a.weights[at + i];
        if (!isfinite(w) || w < 0.0f) flags |= 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.k; i += kGroupThreads) {
        const int r = i % a.k, e = sid[i];
        bool valid = e >= 0 && e < a.E;
        for (int q = 1; q <= r; ++q) valid &= sid[i - q] != e;
        if (!valid) flags |= 1;
        local(i, valid ? atomicAdd(&counts[e], 1) : -1);
    }
    if (flags) atomicOr(a.error, flags);
}
// Exclusive sums over the experts' numbers n(e); base(e, sum) takes them and
// returns the sum with all of the experts up to e, last(sum) the total.
template<class Number, class Base, class Last>
__device__ __forceinline__ void scan_experts(const I8GroupArgs &a, const Number &number, const Base &base, const Last &last) {
    __shared__ int sums[kGroupThreads / 64];
    const int per = (a.Ep + kGroupThreads - 1) / kGroupThreads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lo = min(a.Ep, static_cast<int>(threadIdx.x) * per), hi = min(a.Ep, lo + per);
    int mine = 0;
    for (int e = lo; e < hi; ++e) mine += number(e);
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int run = incl - mine;
    for (int w = 0; w < wave; ++w) run += sums[w];
    for (int e = lo; e < hi; ++e) {
        const int n = number(e);
        base(e, run, n);
        run += n;
        if (e + 1 == a.Ep) last(run);
    }
    __syncthreads();
}
__device__ __forceinline__ void place_route(const I8GroupArgs &a, int i, int place) {
    a.g.place[i] = place;
    if (place >= 0) a.g.token[place] = i / a.k;
}

// Up to kSmallRoutes routes: the first workgroup groups them, the others quantise x.
inline constexpr int kSmallRoutes = 2048;
template<int T, int L, int V>
__global__ __launch_bounds__(kGroupThreads) void k_i8_prepare_small(I8GroupArgs a, I8Rows x) {
    extern __shared__ int32_t group_lds[];
    if (blockIdx.x > 0) {
        quantize_rows<T, L, V>(x, blockIdx.x - 1);
        return;
    }
    int32_t *sid = group_lds, *counts = sid + a.tokens * a.k;
    int number[kSmallRoutes / kGroupThreads];
#pragma unroll
    for (int j = 0; j < kSmallRoutes / kGroupThreads; ++j) number[j] = -1;
    count_routes(a, 0, a.tokens, sid, counts, [&](int i, int n) {
#pragma unroll
        for (int j = 0; j < kSmallRoutes / kGroupThreads; ++j)
            if (i / kGroupThreads == j) number[j] = n;
    });
    __syncthreads();
    // Rows below bit 16 (at most 2,048 routes and as many of the shared expert),
    // groups that have any above.
    const auto number_of = [&](int e) {
        const int n = e < a.E ? counts[e] : a.tokens;
        return n > 0 ? n | 1 << 16 : 0;
    };
    scan_experts(a, number_of, [&](int e, int run, int n) {
        const int first = run & 0xffff;
        counts[e] = first;
        a.g.offsets[e] = first;
        if (n) a.g.active[run >> 16] = make_int4(e, first, n & 0xffff, 0);
    }, [&](int all) {
        a.g.offsets[a.Ep] = all & 0xffff;
        *a.g.groups = all >> 16;
    });
#pragma unroll
    for (int j = 0; j < kSmallRoutes / kGroupThreads; ++j) {
        const int i = j * kGroupThreads + threadIdx.x;
        if (i < a.tokens * a.k) place_route(a, i, number[j] < 0 ? -1 : counts[sid[i]] + number[j]);
    }
    if (a.Ep > a.E)
        for (int t = threadIdx.x; t < a.tokens; t += kGroupThreads) a.g.token[counts[a.E] + t] = t;
}

// More routes: blocks of tokens count theirs (place holds a route's number in its
// block) beside the workgroups that quantise x; then each block sums up the counts
// of those before it.
template<int T, int L, int V>
__global__ __launch_bounds__(kGroupThreads) void k_i8_count(I8GroupArgs a, I8Rows x) {
    extern __shared__ int32_t group_lds[];
    if (static_cast<int>(blockIdx.x) >= a.blocks) {
        quantize_rows<T, L, V>(x, blockIdx.x - a.blocks);
        return;
    }
    const int t0 = blockIdx.x * a.per, n = min(a.per, a.tokens - t0);
    int32_t *counts = group_lds, *sid = counts + a.Ep;
    count_routes(a, t0, n, sid, counts, [&](int i, int number) { a.g.place[static_cast<size_t>(t0) * a.k + i] = number; });
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kGroupThreads) a.g.counts[static_cast<size_t>(blockIdx.x) * a.Ep + e] = counts[e];
}
__global__ __launch_bounds__(kGroupThreads) void k_i8_place(I8GroupArgs a) {
    extern __shared__ int32_t group_lds[];
    int32_t *all = group_lds, *before = all + a.Ep;
    for (int e = threadIdx.x; e < a.Ep; e += kGroupThreads) {
        int n = 0, b = 0;
        if (e < a.E) {
            for (int j0 = 0; j0 < a.blocks; j0 += 16) {
                int c[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) c[i] = a.g.counts[static_cast<size_t>(min(j0 + i, a.blocks - 1)) * a.Ep + e];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    n += j0 + i < a.blocks ? c[i] : 0;
                    b += j0 + i < static_cast<int>(blockIdx.x) ? c[i] : 0;
                }
            }
        } else {
            n = a.tokens;
        }
        all[e] = n;
        before[e] = b;
    }
    __syncthreads();
    const bool writer = blockIdx.x == 0;
    scan_experts(a, [&](int e) { return all[e]; }, [&](int e, int run, int) {
        before[e] += run;
        if (writer) a.g.offsets[e] = run;
    }, [&](int rows) {
        if (writer) a.g.offsets[a.Ep] = rows;
    });
    const int t0 = blockIdx.x * a.per, n = min(a.per, a.tokens - t0);
    const size_t at = static_cast<size_t>(t0) * a.k;
    for (int i = threadIdx.x; i < n * a.k; i += kGroupThreads) {
        const int number = a.g.place[at + i];
        if (number >= 0) place_route(a, static_cast<int>(at) + i, before[a.ids[at + i]] + number);
    }
    if (a.Ep > a.E)
        for (int i = threadIdx.x; i < n; i += kGroupThreads) a.g.token[before[a.E] + t0 + i] = t0 + i;
}

hipError_t launch_prepare_i8(I8GroupArgs a, const I8Rows &x, int type, hipStream_t s) {
    const bool small = a.tokens * a.k <= kSmallRoutes;
    a.per = small ? a.tokens : std::max(64, (a.tokens + 127) / 128);
    a.blocks = (a.tokens + a.per - 1) / a.per;
    const size_t lds = (static_cast<size_t>(a.per) * a.k + a.Ep) * 4;
    with_quantizer(type, x.width, [&](auto t, auto l, auto v) {
        const dim3 grid(a.blocks + quantize_blocks(x.rows, l)), block(kGroupThreads);
        if (small) k_i8_prepare_small<t, l, v><<<grid, block, lds, s>>>(a, x);
        else k_i8_count<t, l, v><<<grid, block, lds, s>>>(a, x);
    });
    hipError_t r = hipGetLastError();
    if (r != hipSuccess || small) return r;
    k_i8_place<<<dim3(a.blocks), dim3(kGroupThreads), static_cast<size_t>(a.Ep) * 8, s>>>(a);
    return hipGetLastError();
}

// ------------------------------------------------------------------- sums ---
inline constexpr int kDownPairs = 33;   // 32 routes and the shared expert
struct I8FoldArgs {
    const float *c;            // [pairs][H] outputs of the experts
    I8Groups g;
    const float *weights, *shared_gate;
    void *y;
    int tokens, H, k, E, shared;
    int *error;
};
// y = +0 + w_0 c_0 + .. in rank order, + sigmoid(gate) shared, with the flags of
// moe_ffn_forward's sum, rounded once: a workgroup a token, V elements (16 bytes of
// the contributions) a thread, eight rows' loads in flight.
template<int T>
__global__ __launch_bounds__(256) void k_i8_fold(I8FoldArgs a) {
    constexpr int V = 4;
    typedef float Row __attribute__((ext_vector_type(4)));
    __shared__ int place[kDownPairs];
    __shared__ float weight[kDownPairs];
    const size_t t = blockIdx.x;
    int flags = 0;
    if (threadIdx.x <= static_cast<unsigned>(a.k)) {
        const int r = threadIdx.x;
        const size_t route = t * a.k + r;
        int at = -1;
        float w = 1.0f;
        if (r < a.k) {
            at = a.g.place[route];
            w = a.weights[route];
            if (at >= 0 && !isfinite(w)) { flags |= 1; w = 0.0f; }
        } else if (a.shared) {
            at = a.g.offsets[a.E] + static_cast<int>(t);
            if (a.shared_gate) {
                float g = a.shared_gate[t];
                if (!isfinite(g)) { flags |= 1; g = 0.0f; }
                w = 1.0f / (1.0f + moe_expf(-g));
                if (!isfinite(w)) { flags |= 2; w = 0.0f; }
            }
        }
        place[r] = at;
        weight[r] = w;
    }
    // A weight that is not finite gives up the routed sum, such a gate all of it.
    const uint64_t first = __builtin_amdgcn_ballot_w64(flags != 0);   // of the first wave, which has them all
    __shared__ uint64_t lost_ranks;
    if (threadIdx.x == 0) lost_ranks = first;
    __syncthreads();
    const uint64_t lost = lost_ranks;
    const bool no_routes = (lost & ((uint64_t{1} << a.k) - 1)) != 0, no_shared = (lost >> a.k & 1) != 0;
    for (int h = threadIdx.x * V; h < a.H; h += 256 * V) {
        const auto load = [&](int r) {
            return __builtin_nontemporal_load(reinterpret_cast<const Row *>(a.c + static_cast<size_t>(place[r]) * a.H + h));
        };
        int f[V] = {};
        float v[V] = {};
        Row shared = {};
        if (a.shared) shared = load(a.k);
        for (int r0 = 0; r0 < a.k; r0 += 8) {
            Row x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (r0 + q < a.k && place[r0 + q] >= 0) x[q] = load(r0 + q);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if (r0 + q >= a.k || place[r0 + q] < 0) continue;
                const float w = weight[r0 + q];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float c = x[q][e];
                    if (!isfinite(c)) { f[e] |= 1; c = 0.0f; }
                    float p = w * c;
                    if (!isfinite(p)) { f[e] |= 2; p = 0.0f; }
                    v[e] = v[e] + p;
                    if (!isfinite(v[e])) { f[e] |= 2; v[e] = 0.0f; }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (f[e] || no_routes) v[e] = 0.0f;
            flags |= f[e];
            if (a.shared) {
                int sf = no_shared ? 1 : 0;
                float c = shared[e];
                if (!isfinite(c)) { sf |= 1; flags |= 1; c = 0.0f; }
                v[e] = v[e] + weight[a.k] * c;
                if (!isfinite(v[e])) { sf |= 2; flags |= 2; v[e] = 0.0f; }
                if (sf) v[e] = 0.0f;
            }
        }
        store4<T>(a.y, t * a.H + h, v);
    }
    if (flags) atomicOr(a.error, flags);
}

// ------------------------------------------- few tokens: gate and up ---
// Work item (group, pair of tiles): 16 rows of gate and of up, whose chunks the eight
// waves share out (wave w: chunks w, w + 8, ..), straight from memory into
// registers, against all of the group's rows, 16 at a time; the sums meet in LDS.
// A workgroup takes items in turn, each with its first tiles on their way before
// the last one's sums are done.  2048/512, 1 / 8 / 32 tokens 8.3 / 28.9 / 84 us: bound by
// three dependent trips to memory (group, its rows' numbers, the rows), then by HBM
// (160 MB at 5.5 TB/s); the grouped products' kernel 14.8 / 32.2 / 81, at 64 tokens 120
// against 129.
struct I8GateUpArgs {
    const uint8_t *blocks;
    const float *sw;
    const int8_t *x;
    const float *sx;
    int64_t pitch;
    I8Groups g;
    float *middle;             // [pairs][I]
    int I, rows, K, chunks;    // rows: 2 i8_rows(I)
    int *error;
};
inline constexpr int kFewTokens = 32;   // tokens up to which gate and up take this kernel
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4))) void k_i8_gate_up_few(I8GateUpArgs a) {
    constexpr int U = 4, W = 8, Most = kFewTokens / 16;   // chunks in flight, waves, row tiles of x
    __shared__ i32x4 red[W][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = i8_rows(a.I) / 16, items = *a.g.groups * pairs;
    uint4 f[U][2];
    const uint8_t *w = a.blocks;
    const auto load = [&](int c0) {
        const auto one = [&](int u) {
            const size_t at = static_cast<size_t>(c0 + u * W) * kI8BlockBytes;
            f[u][0] = load_once(w + at);
            f[u][1] = load_once(w + at + 1024);
        };
        // All at once, without a branch between them; where there are fewer, no others
        // in their place (2560/640, 40 chunks, 8 tokens 88.4 -> 81.1 us a layer).
        if (c0 + (U - 1) * W < a.chunks) {
#pragma unroll
            for (int u = 0; u < U; ++u) one(u);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + u * W < a.chunks) one(u);
        }
    };
    const auto select = [&](int item) {
        const int4 group = a.g.active[item / pairs];
        const int pair = item % pairs, e = __builtin_amdgcn_readfirstlane(group.x);
        w = a.blocks + (static_cast<size_t>(e) * (a.rows / kI8Block) + pair / 2) * a.chunks * kI8BlockBytes + (pair & 1) * 2048 + lane * 16;
        load(wave);
        return make_int4(e, __builtin_amdgcn_readfirstlane(group.y), __builtin_amdgcn_readfirstlane(group.z), pair);
    };
    int flags = 0;
    int4 next = static_cast<int>(blockIdx.x) < items ? select(blockIdx.x) : int4{};
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int4 now = next;   // expert, first place, rows, pair
        const int tiles = (now.z + 15) / 16;
        const int8_t *x[Most];
#pragma unroll
        for (int t = 0; t < Most; ++t) {
            const int n = min(t * 16 + (lane & 15), now.z - 1);
            x[t] = a.x + static_cast<int64_t>(t < tiles ? a.g.token[now.y + n] : 0) * a.pitch + (lane >> 4) * 16;
        }
        i32x4 acc[Most][2];
#pragma unroll
        for (int t = 0; t < Most; ++t) acc[t][0] = acc[t][1] = i32x4{0, 0, 0, 0};
        for (int c0 = wave; c0 < a.chunks; c0 += W * U) {
            if (c0 != wave) load(c0);
#pragma unroll
            for (int t = 0; t < Most; ++t) {
                if (t >= tiles) break;
                uint4 v[U];
                const auto part = [&](int u) {
                    const int c = c0 + u * W;
                    v[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (c * kI8Chunk + (lane >> 4) * 16 < a.K) v[u] = *reinterpret_cast<const uint4 *>(x[t] + c * kI8Chunk);
                };
                if (c0 + (U - 1) * W < a.chunks) {
#pragma unroll
                    for (int u = 0; u < U; ++u) part(u);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c0 + u * W < a.chunks) part(u);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (c0 + u * W >= a.chunks) break;
                    acc[t][0] = i8_dot(f[u][0], v[u], acc[t][0]);
                    acc[t][1] = i8_dot(f[u][1], v[u], acc[t][1]);
                }
            }
        }
        if (item + static_cast<int>(gridDim.x) < items) next = select(item + gridDim.x);
#pragma unroll
        for (int t = 0; t < Most; ++t) {
            if (t >= tiles) break;
            red[wave][0][lane] = acc[t][0];
            red[wave][1][lane] = acc[t][1];
            __syncthreads();
            // Thread i < 256: result i % 4 of lane i / 4.
            if (threadIdx.x < 256) {
                const int l = threadIdx.x >> 2, q = threadIdx.x & 3, n = t * 16 + (l & 15), j = now.w * 16 + (l >> 4) * 4 + q;
                int g = 0, u = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    g += reinterpret_cast<const int *>(&red[i][0][l])[q];
                    u += reinterpret_cast<const int *>(&red[i][1][l])[q];
                }
                if (n < now.z && j < a.I) {
                    const float sx = a.sx[a.g.token[now.y + n]];
                    const float *s = a.sw + static_cast<size_t>(now.x) * a.rows + (now.w >> 2) * 128 + (now.w & 3) * 16 + (l >> 4) * 4 + q;
                    a.middle[static_cast<size_t>(now.y + n) * a.I + j] =
                        silu_product(static_cast<float>(g) * (sx * s[0]), static_cast<float>(u) * (sx * s[64]), flags);
                }
            }
            __syncthreads();
        }
    }
    if (flags) atomicOr(a.error, flags);
}

// ----------------- few tokens an expert (down_in_one): down and the sum in one ---
// Workgroup (t, slice of `tiles` tiles of 16 rows); wave w takes ranks w, w + W, ..
// It quantises the rank's middle row into LDS in pieces of eight chunks and streams
// the expert's tiles past it, a tile's chunks of a piece at a time with the next
// tile's on their way.  All 16 columns of its MFMA hold the one token.
struct I8DownArgs {
    const uint8_t *blocks;     // [E'][H / 64][chunks]
    const float *sw;           // [E'][rows]
    const float *middle;       // [pairs][I]
    const int32_t *ids;
    I8Groups g;
    const float *weights, *shared_gate;
    void *y;
    int T, H, I, E, k, P1;     // P1 = k + shared
    int rows, chunks;
    int *error;
};
inline constexpr int kDownPiece = 8, kDownTiles = 16;
template<int Y>
__global__ __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(4))) void k_i8_down_fold(I8DownArgs a, int tiles) {
    extern __shared__ __attribute__((aligned(16))) int part[];   // [rank][16 tiles]: sums, then outputs
    __shared__ __attribute__((aligned(16))) uint8_t codes[16][kDownPiece * kI8Chunk];
    __shared__ float weight[kDownPairs];
    __shared__ int valid[kDownPairs];
    const int R = 16 * tiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    // Workgroup i runs on XCD i % 8: all tokens of one slice on one XCD, one after the
    // other, so that experts they share come from its L2.
    const int row_tiles = a.rows / 16, S = (row_tiles + tiles - 1) / tiles;
    const int j = blockIdx.x >> 3, t = j % a.T, s = (blockIdx.x & 7) + 8 * (j / a.T);
    if (s >= S) return;
    const int tile0 = s * tiles, here = min(tiles, row_tiles - tile0);
    for (int r = wave; r < a.P1; r += W) {
        const int place = r < a.k ? a.g.place[t * a.k + r] : a.g.offsets[a.E] + t;
        const int e = r < a.k ? a.ids[t * a.k + r] : a.E;
        if (lane == 0) {
            weight[r] = r < a.k ? a.weights[t * a.k + r] : a.shared_gate ? a.shared_gate[t] : 1.0f;
            valid[r] = place >= 0;
        }
        const int at = __builtin_amdgcn_readfirstlane(place), expert = __builtin_amdgcn_readfirstlane(e);
        if (at < 0) continue;
        const float *mid = a.middle + static_cast<size_t>(at) * a.I;
        const uint8_t *w = a.blocks + static_cast<size_t>(expert) * a.rows / kI8Block * a.chunks * kI8BlockBytes;
        const float *sw = a.sw + static_cast<size_t>(expert) * a.rows;
        uint4 f[2][kDownPiece];
        // Tile n's chunks k0 .. + kb - 1.
        const auto load = [&](int n, int k0, int kb, uint4 (&to)[kDownPiece]) {
            const int tile = tile0 + min(n, here - 1);
            const uint4 *p = reinterpret_cast<const uint4 *>(w + (static_cast<size_t>(tile >> 2) * a.chunks + k0) * kI8BlockBytes + (tile & 3) * 1024) + lane;
#pragma unroll
            for (int u = 0; u < kDownPiece; ++u) to[u] = p[min(u, kb - 1) * (kI8BlockBytes / 16)];   // past the piece: the last again, not used
        };
        load(0, 0, min(kDownPiece, a.chunks), f[0]);
        uint32_t m = 0;
        for (int c = lane * 8; c < a.I; c += 512) {
            float v[8];
            unpack8<kF32>(load8_raw<kF32>(mid, c), v);
#pragma unroll
            for (int q = 0; q < 8; ++q) m = max(m, magnitude(v[q]));
        }
        const GroupScale scale = row_scale(wave_max(m));
        for (int k0 = 0; k0 < a.chunks; k0 += kDownPiece) {
            const int kb = min(kDownPiece, a.chunks - k0), col = k0 * kI8Chunk + lane * 8;
            if (k0 > 0) load(0, k0, kb, f[0]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last piece's reads are done
            Raw8 raw{};
            if (col < a.I) raw = load8_raw<kF32>(mid, col);
            float v[8];
            unpack8<kF32>(raw, v);
            *reinterpret_cast<uint2 *>(&codes[wave][lane * 8]) = quantize8_i8(v, scale);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            uint4 x[kDownPiece];
#pragma unroll
            for (int u = 0; u < kDownPiece; ++u) x[u] = *reinterpret_cast<const uint4 *>(&codes[wave][u * kI8Chunk + (lane >> 4) * 16]);
            const auto multiply = [&](int n, const uint4 (&from)[kDownPiece]) {
                const int tile = tile0 + n, row = n * 16 + (lane >> 4) * 4;
                i32x4 *out = reinterpret_cast<i32x4 *>(&part[r * R + row]);
                i32x4 acc = k0 > 0 ? *out : i32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < kDownPiece; ++u)
                    if (u < kb) acc = i8_dot(from[u], x[u], acc);
                if (k0 + kDownPiece >= a.chunks) {
                    const float *c = sw + (tile >> 1) * 32 + (lane >> 4) * 8 + (tile & 1) * 4;
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[q] = __float_as_int(static_cast<float>(acc[q]) * (scale.s * c[q]));
                }
                if ((lane & 15) == 0) *out = acc;
            };
            for (int n = 0; n < here; n += 2) {
                load(n + 1, k0, kb, f[1]);
                multiply(n, f[0]);
                if (n + 1 >= here) break;
                load(n + 2, k0, kb, f[0]);
                multiply(n + 1, f[1]);
            }
        }
    }
    __syncthreads();
    int flags = 0;
    for (int i = threadIdx.x; i < here * 16; i += blockDim.x) {
        const int tile = tile0 + (i >> 4), row = (tile >> 1) * 32 + (i >> 2 & 3) * 8 + (tile & 1) * 4 + (i & 3);
        if (row >= a.H) continue;
        const float v = fold(a.k, a.P1 > a.k, a.shared_gate != nullptr, valid, weight, [&](int r) { return __int_as_float(part[r * R + i]); }, flags);
        store1<Y>(a.y, static_cast<size_t>(t) * a.H + row, v);
    }
    if (flags) atomicOr(a.error, flags);
}

hipError_t launch_down_fold(const I8DownArgs &a, int type, hipStream_t s) {
    const int row_tiles = a.rows / 16;
    // Row tiles a workgroup: the fewest on the busiest CU, and of such choices the one
    // with the fewest workgroups a CU (one / two / four first, us a layer of 2048/512:
    // 4 tokens 33.2 / 37.5 / 37.3, 8 52.0 / 54.5 / 62.1).
    int tiles = 1, best = 1 << 30, fewest = 0;
    for (int n = 1; n <= kDownTiles; ++n) {
        const int rounds = (a.T * ((row_tiles + n - 1) / n) + 255) / 256;
        if (rounds * n < best || (rounds * n == best && rounds < fewest)) {
            tiles = n;
            best = rounds * n;
            fewest = rounds;
        }
    }
    const dim3 grid(static_cast<unsigned>((row_tiles + tiles - 1) / tiles + 7) / 8 * 8 * a.T), block(64 * std::min(16, a.P1));
    const size_t lds = static_cast<size_t>(a.P1) * tiles * 64;
    if (type == kF32) k_i8_down_fold<kF32><<<grid, block, lds, s>>>(a, tiles);
    else if (type == kBF16) k_i8_down_fold<kBF16><<<grid, block, lds, s>>>(a, tiles);
    else k_i8_down_fold<kF16><<<grid, block, lds, s>>>(a, tiles);
    return hipGetLastError();
}

}  // namespace
}  // namespace moe

// ------------------------------------------------------------------ C ABI ---
struct moe_i8_bank {
    int experts = 0, input = 0, output = 0, device = 0;
    uint8_t *mem = nullptr;   // blocks, scales
    float *scales = nullptr;
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
    float *middle = nullptr;                       // [pairs][I]
    float *contrib = nullptr;                      // [pairs][H]
    int *dropped = nullptr;                        // flags of rows that are not used
    moe::I8Groups groups{};
};

namespace {

constexpr int kInvalid = hipErrorInvalidValue;

bool aligned(const void *p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t round_up(size_t v, size_t m) { return (v + m - 1) / m * m; }
bool is_type(int t) { return t == MOE_F32 || t == MOE_BF16 || t == MOE_F16; }
int64_t odd_pitch(int width) { return static_cast<int64_t>(moe::i8_chunks(width) | 1) * moe::kI8Chunk; }
size_t block_bytes(int rows, int cols) { return static_cast<size_t>(moe::i8_rows(rows)) * moe::i8_chunks(cols) * moe::kI8Chunk; }

// `count` matrices on the host or the device into blocks and scales.
hipError_t upload(const moe_i8_matrix &m, uint8_t *to, float *scales, size_t count, int rows, int cols, int part, bool on_device) {
    const size_t bytes = count * rows * cols;
    const int8_t *codes = static_cast<const int8_t *>(m.codes);
    void *staging = nullptr;
    hipError_t r = hipSuccess;
    if (!on_device) {
        if ((r = hipMalloc(&staging, bytes)) != hipSuccess) return r;
        r = hipMemcpy(staging, m.codes, bytes, hipMemcpyHostToDevice);
        codes = static_cast<const int8_t *>(staging);
    }
    if (r == hipSuccess) r = moe::launch_i8_repack(codes, to, count, rows, cols, part, nullptr);
    const hipMemcpyKind kind = on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice;
    const size_t width = static_cast<size_t>(rows) * 4, padded = static_cast<size_t>(moe::i8_rows(rows)) * 4;
    if (part == moe::kI8Whole) {
        if (r == hipSuccess) r = hipMemcpy2D(scales, padded, m.scales, width, width, count, kind);
    } else if (rows % 64 == 0) {
        // 64 of gate, 64 of up in turn.
        if (r == hipSuccess) r = hipMemcpy2D(scales + part * 64, 512, m.scales, 256, 256, count * (rows / 64), kind);
    } else {
        for (int at = 0; at < rows && r == hipSuccess; at += 64)
            r = hipMemcpy2D(scales + at * 2 + part * 64, 2 * padded, m.scales + at, width, std::min(64, rows - at) * 4, count, kind);
    }
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

// Down and the sum in one launch, which reads an expert again, from L2, for each of its
// tokens, or down grouped by expert, in three.  The first where what it reads again
// of the routed experts is less than 100 MB of an evenly routed batch (the shared one's
// reads are cheap: all tokens' are near each other); us a layer, one launch / three:
//   2048/512, top-10 of 512      16 tokens 88.3 / 106   24 122 / 136   32 148 / 150   48 183 / 176
//   2048/768, top-8 of 128       16        91.0 / 96.3  24 118 / 109   32 123 / 117   48 139 / 118
//   2048/1024, top-6 of 64       16        71.9 / 76.0  24 95.8 / 87.4 32 92.7 / 86.7 48 108 / 84.8
//   4096/2048, top-2 of 8         8        49.9 / 53.6  16 61.6 / 55.7 32 65.6 / 56.2 48 70.7 / 55.5
//   2048/512, top-2 of 8          8        16.1 / 23.0  16 18.6 / 23.2 48 25.5 / 27.8 64 29.2 / 28.2
// Up to 64 tokens, where three launches have caught up on every shape above.
inline constexpr int kFewDown = 64;
bool down_in_one(const moe_i8_layer_config &c, int tokens) {
    const double E = c.experts, pairs = static_cast<double>(tokens) * c.top_k;
    const double reached = E * (1.0 - std::pow(1.0 - c.top_k / E, tokens));
    return tokens <= kFewDown && (pairs - reached) * c.hidden * c.intermediate <= 100e6;
}

struct LayerLayout {
    size_t gate_up, down, gate_up_s, down_s, weights;   // offsets and end of the weights
    size_t x, x_s, m, m_s, middle, contrib, offsets, token, place, counts, active, groups, dropped, workspace;
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
    const size_t P = T * (c.top_k + c.has_shared);
    l.gate_up = take(Ep * 2 * block_bytes(c.intermediate, c.hidden));
    l.down = take(Ep * block_bytes(c.hidden, c.intermediate));
    l.gate_up_s = take(Ep * 2 * moe::i8_rows(c.intermediate) * 4);
    l.down_s = take(Ep * moe::i8_rows(c.hidden) * 4);
    l.weights = at;
    at = 0;
    l.x = take(T * odd_pitch(c.hidden));
    l.x_s = take(T * 4);
    l.m = take(P * odd_pitch(c.intermediate));
    l.m_s = take(P * 4);
    l.middle = take(P * I * 4);
    l.contrib = take(P * H * 4);
    l.offsets = take((Ep + 1) * 4);
    l.token = take(P * 4);
    l.place = take(T * c.top_k * 4);
    l.counts = take(std::min<size_t>(128, (T + 63) / 64) * Ep * 4);
    l.active = take(Ep * 16);
    l.groups = take(4);
    l.dropped = take(4);
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
    const size_t scale_at = block_bytes(output, input) * experts, scale_bytes = static_cast<size_t>(experts) * moe::i8_rows(output) * 4;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&B->mem, scale_at + scale_bytes);
    B->scales = reinterpret_cast<float *>(B->mem + scale_at);
    if (r == hipSuccess)
        r = upload(moe_i8_matrix{codes, scales}, B->mem, B->scales, experts, output, input, moe::kI8Whole, weights_on_device != 0);
    if (r != hipSuccess) { release(B); return r; }
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
    a.blocks = B->mem;
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
    a.rows = moe::i8_rows(B->output);
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
    const size_t E = c->experts;
    // Weights that another stream is still writing are complete after this.
    hipError_t r = hipDeviceSynchronize();
    if (r == hipSuccess) r = hipMalloc(&L->mem, l.weights);
    if (r == hipSuccess) r = hipMalloc(&L->ws, l.workspace);
    const auto bank = [&](const moe_i8_matrix *m, size_t at, size_t count) {
        uint8_t *gate_up = L->mem + l.gate_up + at * 2 * block_bytes(I, H), *down = L->mem + l.down + at * block_bytes(H, I);
        float *gate_up_s = reinterpret_cast<float *>(L->mem + l.gate_up_s) + at * 2 * moe::i8_rows(I);
        float *down_s = reinterpret_cast<float *>(L->mem + l.down_s) + at * moe::i8_rows(H);
        if (r == hipSuccess) r = upload(m[0], gate_up, gate_up_s, count, I, H, moe::kI8Gate, on_device);
        if (r == hipSuccess) r = upload(m[1], gate_up, gate_up_s, count, I, H, moe::kI8Up, on_device);
        if (r == hipSuccess) r = upload(m[2], down, down_s, count, H, I, moe::kI8Whole, on_device);
    };
    if (r == hipSuccess) bank(experts, 0, E);
    if (r == hipSuccess && c->has_shared) bank(shared, E, 1);
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
    L->groups = moe::I8Groups{ints(l.offsets), ints(l.token), ints(l.place), ints(l.counts),
                              reinterpret_cast<int4 *>(L->ws + l.active), ints(l.groups)};
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
    const moe::I8GroupArgs ga{ids, weights, L->groups, tokens, c.top_k, c.experts, Ep, 0, 0, error};
    const moe::I8Rows xr{x, c.hidden, c.hidden, static_cast<size_t>(tokens), L->x, L->x_pitch, L->x_s, error};
    hipError_t r = moe::launch_prepare_i8(ga, xr, type, s);
    if (r != hipSuccess) return r;
    moe::I8Args a{};
    a.blocks = L->gate_up;
    a.sw = L->gate_up_s;
    a.x = L->x;
    a.sx = L->x_s;
    a.pitch = L->x_pitch;
    a.index = L->groups.token;
    a.x_rows = tokens;
    a.offsets = L->groups.offsets;
    a.experts = Ep;
    a.y = L->middle;
    a.y_stride = c.intermediate;
    a.M = c.intermediate;
    a.rows = 2 * moe::i8_rows(c.intermediate);
    a.N = pairs;
    a.K = c.hidden;
    a.chunks = moe::i8_chunks(c.hidden);
    a.error = error;
    if (tokens <= moe::kFewTokens) {
        const moe::I8GateUpArgs u{a.blocks, a.sw, a.x, a.sx, a.pitch, L->groups, L->middle, a.M, a.rows, a.K, a.chunks, error};
        const size_t items = static_cast<size_t>(std::min(tokens * c.top_k, c.experts) + c.has_shared) * (moe::i8_rows(a.M) / 16);   // at most
        moe::k_i8_gate_up_few<<<dim3(static_cast<unsigned>(std::min<size_t>(items, 512))), dim3(512), 0, s>>>(u);
        r = hipGetLastError();
    } else {
        r = moe::launch_grouped<moe::kStoreMiddle, moe::kF32>(a, s);
    }
    if (r != hipSuccess) return r;
    if (down_in_one(c, tokens)) {
        const moe::I8DownArgs d{L->down, L->down_s, L->middle, ids, L->groups, weights, shared_gate, y, tokens, c.hidden,
                                c.intermediate, c.experts, c.top_k, c.top_k + c.has_shared, moe::i8_rows(c.hidden),
                                moe::i8_chunks(c.intermediate), error};
        return moe::launch_down_fold(d, type, s);
    }
    // Rows that no group took (dropped routes) are quantised as well, and not used;
    // what they hold raises no flag of this call, and SiLU(g) u is always finite.
    const moe::I8Rows mr{L->middle, c.intermediate, c.intermediate, static_cast<size_t>(pairs), L->m, L->m_pitch, L->m_s, L->dropped};
    if ((r = moe::launch_quantize_i8(mr, moe::kF32, s)) != hipSuccess) return r;
    a.blocks = L->down;
    a.sw = L->down_s;
    a.x = L->m;
    a.sx = L->m_s;
    a.pitch = L->m_pitch;
    a.index = nullptr;
    a.x_rows = pairs;
    a.y = L->contrib;
    a.y_stride = c.hidden;
    a.M = c.hidden;
    a.rows = moe::i8_rows(c.hidden);
    a.K = c.intermediate;
    a.chunks = moe::i8_chunks(c.intermediate);
    if ((r = moe::launch_grouped<moe::kStoreRows, moe::kF32>(a, s)) != hipSuccess) return r;
    const moe::I8FoldArgs f{L->contrib, L->groups, weights, shared_gate, y, tokens, c.hidden, c.top_k, c.experts, c.has_shared, error};
    const dim3 grid(tokens), block(256);
    if (type == MOE_F32) moe::k_i8_fold<moe::kF32><<<grid, block, 0, s>>>(f);
    else if (type == MOE_BF16) moe::k_i8_fold<moe::kBF16><<<grid, block, 0, s>>>(f);
    else moe::k_i8_fold<moe::kF16><<<grid, block, 0, s>>>(f);
    return hipGetLastError();
}

}  // extern "C"
