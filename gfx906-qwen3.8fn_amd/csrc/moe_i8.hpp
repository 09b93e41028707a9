// The 8-bit integer operators: int8 matrices with one fp32 scale per output
// channel, int8 activations with one per row.  gfx950 (CDNA4), wave64.
//   y[n][m] = (sum_k cx[n][k] cw[m][k]) * (sx[n] * sw[m])
// The sum is a whole number that int32 holds (2^28 at most: K <= 16384), so its
// order, the tile and the number of waves that share K change no bit of y.
//
// Matrix layout.  A matrix [M][K] is kept in blocks of 64 rows x 64 columns (4
// KiB, zero past its edges), [ceil(M/64)][ceil(K/64)], each as four tiles of 16
// rows in the order in which a wave's lanes take them as an operand of
// v_mfma_i32_16x16x64_i8: lane l holds tile row l % 16, columns 16 (l / 16) .. +
// 15.  The product leaves rows 4 g .. + 3 of a tile in lanes 16 g .. + 15; row 4 g +
// q of tile i is row 32 (i / 2) + 8 g + 4 (i % 2) + q of the block, so that a lane's
// results of two tiles are eight neighbours in a row of y and a store of 16-bit
// ones fills 64 bytes of each row; with 16 neighbours in a lane, and stores that fill
// every other 16 bytes, 2048 x 2048 at 1,032 fp32 rows took 19.8 us instead of 18.1.
// What a product reads past a row of activations meets the zeros past the matrix
// row, so rows need no padding.
//
// Gate and up matrices of an expert lie together as one of 2 I rows (I rounded up
// to 64), in which 64 rows of both make two blocks: tile 2 i holds rows 16 i .. + 15
// of gate, tile 2 i + 1 those of up.
#pragma once

#include "moe_fp8.hpp"   // element types, loads into LDS

#include <type_traits>

namespace moe {

inline constexpr int kI8Block = 64, kI8Chunk = 64, kI8BlockBytes = kI8Block * kI8Chunk;
__host__ __device__ constexpr int i8_chunks(int cols) { return (cols + kI8Chunk - 1) / kI8Chunk; }
__host__ __device__ constexpr int i8_rows(int rows) { return (rows + kI8Block - 1) / kI8Block * kI8Block; }

// Canonical int8 codes [matrices][rows][cols] -> blocks.  part: kI8Whole, or the half of a
// pair of gate and up.
enum { kI8Whole = -1, kI8Gate = 0, kI8Up = 1 };
hipError_t launch_i8_repack(const int8_t *codes, uint8_t *blocks, size_t matrices, int rows, int cols, int part,
                            hipStream_t s);
// Rows x [rows][width] -> codes [rows][pitch], scales [rows].
struct I8Rows {
    const void *x;
    int64_t stride;
    int width;
    size_t rows;
    int8_t *codes;
    int64_t pitch;
    float *scales;
    int *error;
};
hipError_t launch_quantize_i8(const I8Rows &r, int type, hipStream_t s);

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The scale of a row whose largest magnitude has the bits `amax`, as
// group_scale's of e4m3: a = max(|x|max, 2^-100), s = a / 127, r = 127 / a, codes
// rint(x * r).  |x * r| < 127.5, so no code leaves -127 .. 127.
__device__ __forceinline__ GroupScale row_scale(uint32_t amax) {
    const bool bad = amax >= 0x7f800000u;
    const float a = fmaxf(__uint_as_float(bad ? 0u : amax), 0x1p-100f);
    return GroupScale{bad ? 0.0f : a / 127.0f, 127.0f / a, bad};
}
__device__ __forceinline__ uint32_t pack_i8(float a, float b, float c, float d) {
    const auto code = [](float v) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v))); };
    const uint32_t lo = __builtin_amdgcn_perm(code(b), code(a), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(code(d), code(c), 0x04000c0cu);
    return lo | hi;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t m) {
    m = max(m, static_cast<uint32_t>(lane_xor<1>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<2>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<4>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<8>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<16>(static_cast<int>(m))));
    return max(m, static_cast<uint32_t>(lane_xor<32>(static_cast<int>(m))));
}
__device__ __forceinline__ uint2 quantize8_i8(const float (&v)[8], const GroupScale &s) {
    if (s.bad) return make_uint2(0u, 0u);
    return make_uint2(pack_i8(v[0] * s.r, v[1] * s.r, v[2] * s.r, v[3] * s.r),
                      pack_i8(v[4] * s.r, v[5] * s.r, v[6] * s.r, v[7] * s.r));
}

// A row's elements stay in the registers of its L lanes (a wave, or the whole
// workgroup), V times eight of them a lane, between the maximum and the codes:
// bound by memory (16,384 rows of 8,192 bf16 elements 71.5 us, 5.6 TB/s).  block: of
// 256 threads.
template<int T, int L, int V>
__device__ __forceinline__ void quantize_rows(const I8Rows &r, int block) {
    const size_t n = static_cast<size_t>(block) * (256 / L) + threadIdx.x / L;
    const int l = threadIdx.x % L;
    const bool there = n < r.rows;   // whole waves
    Raw8 raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = (i * L + l) * 8;
        raw[i] = load8_any<T>(r.x, (there ? n : 0) * static_cast<size_t>(r.stride) + k, there ? r.width - k : 0);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float v[8];
        unpack8<T>(raw[i], v);
#pragma unroll
        for (int q = 0; q < 8; ++q) m = max(m, magnitude(v[q]));
    }
    m = wave_max(m);
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
        if (k >= r.width) break;
        float v[8];
        unpack8<T>(raw[i], v);
        const uint2 c = quantize8_i8(v, s);
        int8_t *out = r.codes + n * static_cast<size_t>(r.pitch) + k;
        if (k + 8 <= r.width) {
            __builtin_memcpy(out, &c, 8);
        } else {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (k + q < r.width) out[q] = static_cast<int8_t>((q < 4 ? c.x : c.y) >> (8 * (q & 3)));
        }
    }
    if (l == 0) {
        r.scales[n] = s.s;
        if (s.bad) atomicOr(r.error, 1);
    }
}
inline unsigned quantize_blocks(size_t rows, int lanes) {
    const size_t per = 256 / lanes;
    return static_cast<unsigned>((rows + per - 1) / per);
}
// call(T, L, V) as constants for rows of a type and width.
template<class Call>
void with_quantizer(int type, int width, const Call &call) {
    const auto sized = [&](auto t) {
        const auto c = [&](auto l, auto v) { call(t, l, v); };
        if (width <= 512) c(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
        else if (width <= 1024) c(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
        else if (width <= 2048) c(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
        else if (width <= 4096) c(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
        else if (width <= 8192) c(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
        else c(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
    };
    if (type == kF32) sized(std::integral_constant<int, kF32>{});
    else if (type == kBF16) sized(std::integral_constant<int, kBF16>{});
    else sized(std::integral_constant<int, kF16>{});
}

// load_to_lds for what is read once: it leaves the L2 to the rest.
__device__ __forceinline__ void load_to_lds_nt(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                 :: "s"(lds), "v"(off), "s"(r) : "memory", "m0");
}

// 16 bytes that are read once.
__device__ __forceinline__ uint4 load_once(const void *p) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(static_cast<const u32x4 *>(p)));
}

// One tile's products onto acc: lane l has rows 4 (l / 16) + i of the tile against
// token l % 16.
__device__ __forceinline__ i32x4 i8_dot(const uint4 &w, const uint4 &x, const i32x4 &acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), acc, 0, 0, 0);
}

// SiLU(g) * u by the hardware's exponential and reciprocal (8 half ulps): with the Q4
// layers' exact expf, whose table lies in memory, 4,096 tokens of 2048/512 take 615
// us instead of 571, and y is as far from 64 bits (what middle codes on the border
// between two values add to it: 6.7e-5 of its norm, with this 6.5e-5).  0, with a flag, where it is not finite: bit 1 where g or u is
// not, bit 2 where their product is not.
__device__ __forceinline__ float silu_product(float g, float u, int &flags) {
    const float v = g * sigmoid(g) * u;
    if (isfinite(v)) return v;
    flags |= isfinite(g) && isfinite(u) ? 2 : 1;
    return 0.0f;
}

// What a product writes: rows of y, or SiLU(gate) * up in fp32 from pairs of gate and up.
enum { kStoreRows = 0, kStoreMiddle = 1 };

struct I8Args {
    const uint8_t *blocks;    // [experts][rows / 64][chunks] blocks
    const float *sw;          // [experts][rows]; pairs: 64 of gate and 64 of up in turn
    const int8_t *x;          // rows [..][pitch]
    const float *sx;
    int64_t pitch;
    const int32_t *index;     // row of x of each row of the product, or null: the same
    int x_rows;               // rows of x
    const int32_t *offsets;   // [experts + 1]: rows of each expert's matrix; unused where one matrix takes all rows
    int experts;
    void *y;                  // rows of y_type, y_stride apart; kStoreMiddle: fp32
    int64_t y_stride;
    int M, N, K, chunks;      // results in a row (kStoreMiddle: of either half), rows of the product
    int rows;                 // of the blocks: i8_rows(M), twice that for pairs
    int tiles_m;
    int *error;
};

// A work item: rows m0 .. of expert e's matrix, rows r .. r + cols - 1 of the product.
struct I8Item {
    int e, m0, r, cols;
    bool once;   // no other item reads these rows of the matrix
};

// A workgroup of WR x WC waves takes items of 16 TM WR rows of a matrix and 16 TN WC
// rows of x, one after the other, and steps through K in stages of KS chunks, the
// next stages' operands on the way to a ring of S buffers in LDS and the next
// chunk's from there to registers.  The stages of successive items form one
// stream: while an item's results are written, the next one's first stages are on
// their way.  A barrier a stage, with the products of the stage's last chunk still
// to be issued behind it: their operands are in registers, so the barrier and the
// LDS reads after it cost the matrix cores nothing.
//
// The rows' and channels' scales come with an item's first stage into a ring of
// their own, and so do, one item ahead, the indices of its rows: nothing but
// loads into LDS is in flight, and a wait for one of them waits for no later one.
template<int WR, int WC, int TM, int TN, int S, int KS, int Form, int Y, bool Grouped>
struct I8Stream {
    static constexpr int Bytes = elem_bytes(Y);
    static constexpr int W = WR * WC, BM = 16 * TM * WR, BN = 16 * TN * WC;
    static constexpr int ATiles = BM / 16, BTiles = BN / 16;
    static constexpr int ABytes = ATiles * KS * 1024, Stage = ABytes + BTiles * KS * 1024;
    static constexpr int ALoads = ATiles * KS / W, BLoads = BTiles * KS / W, Loads = ALoads + BLoads;   // of a wave and stage
    static constexpr int PA = Form == kStoreMiddle && BM < 128 ? 128 : BM, PB = (BN + 63) / 64 * 64;      // scales of an item
    static constexpr int Params = (PA + PB) * 4, ParamRing = S + 1;   // items between a load and the end of its use
    static constexpr int Index = Grouped ? PB * 4 * W : 0;   // every wave has its own copy
    static constexpr int Lds = S * Stage + ParamRing * Params + 2 * Index;
    static_assert(S >= 3 && ATiles * KS % W == 0 && BTiles * KS % W == 0 && BM % 64 == 0, "every wave issues the same loads");
    static_assert(4 % TM == 0 || TM % 4 == 0);
    static constexpr uint32_t kPastEnd = 0xc0000000u;   // past every resource here, and no sum with it wraps

    const I8Args &a;
    const uint8_t *lds;
    int lane, wave, wr, wc;
    uint32_t lds0, bread;
    // Of the item whose stages are being loaded.
    __amdgpu_buffer_rsrc_t ar, br;
    uint32_t aoff, boff[BLoads];
    bool once;
    int flags = 0;

    __device__ __forceinline__ I8Stream(const I8Args &args, const uint8_t *buffers) : a(args), lds(buffers) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wr = wave / WC;
        wc = wave % WC;
        lds0 = lds_offset(lds);
        // Fragment of row l % 16, piece l / 16, in the permuted order.
        bread = (lane & 15) * 64 + ((lane >> 4) ^ (lane >> 1 & 3)) * 16;
    }
    // Load i of a stage's rows of x: 16 rows of 64 bytes, each row's four pieces
    // permuted by its index so that the fragment reads spread over the LDS banks.
    __device__ __forceinline__ int load_row(int i) const { return (i * W + wave) % BTiles * 16 + (lane >> 2); }
    __device__ __forceinline__ int load_chunk(int i) const { return (i * W + wave) / BTiles; }
    __device__ __forceinline__ uint32_t params_at(int item) const { return S * Stage + item % ParamRing * Params; }
    __device__ __forceinline__ uint32_t index_at(int item) const {
        return S * Stage + ParamRing * Params + ((item & 1) * W + wave) * (PB * 4);
    }
    // Start the loads of an item's row indices; number: of the item, in this workgroup.
    __device__ __forceinline__ void load_index(const I8Item &t, int number) const {
        if (!Grouped || !a.index) return;
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(a.index + t.r, static_cast<uint32_t>(t.cols) * 4);
#pragma unroll
        for (int i = 0; i < PB / 64; ++i) load_word_to_lds(r, (i * 64 + lane) * 4, lds0 + index_at(number) + i * 256);   // 0 past the end
    }
    // Make t the item being loaded; its indices have arrived.  Starts its scales.
    __device__ __forceinline__ void start(const I8Item &t, int number) {
        const uint32_t block_row = static_cast<uint32_t>(a.chunks) * kI8BlockBytes;   // bytes of 64 rows
        ar = buffer_rsrc(a.blocks + (static_cast<size_t>(t.e) * a.rows + t.m0) / kI8Block * block_row,
                         static_cast<uint32_t>(min(a.rows - t.m0, BM) / kI8Block) * block_row);
        aoff = lane * 16;
        once = t.once;
        const bool gather = Grouped && a.index;
        const uint32_t *index = reinterpret_cast<const uint32_t *>(lds + index_at(number));
        if (gather) br = buffer_rsrc(a.x, static_cast<uint32_t>((static_cast<size_t>(a.x_rows) - 1) * a.pitch + a.K));
        else
            br = buffer_rsrc(a.x + static_cast<size_t>(t.r) * a.pitch, static_cast<uint32_t>(static_cast<size_t>(t.cols - 1) * a.pitch + a.K));
        const int piece = (lane & 3) ^ (lane >> 3 & 3);
#pragma unroll
        for (int i = 0; i < BLoads; ++i) {
            const int n = load_row(i);
            uint32_t row = static_cast<uint32_t>(n);
            if (gather) row = index[n];
            const bool there = n < t.cols && (!gather || row < static_cast<uint32_t>(a.x_rows));
            if (n < t.cols && !there) flags |= 1;
            boff[i] = there ? row * static_cast<uint32_t>(a.pitch) + load_chunk(i) * kI8Chunk + piece * 16 : kPastEnd;
        }
        // Scales: wave w loads 64 of them at w, w + W, ..
        const uint32_t to = lds0 + params_at(number);
        const int m0 = Form == kStoreMiddle ? t.m0 / 128 * 128 : t.m0;
        const __amdgpu_buffer_rsrc_t wr_ = buffer_rsrc(a.sw + static_cast<size_t>(t.e) * a.rows + m0, static_cast<uint32_t>(min(a.rows - m0, PA)) * 4);
        const __amdgpu_buffer_rsrc_t xr = gather ? buffer_rsrc(a.sx, static_cast<uint32_t>(a.x_rows) * 4)
                                                 : buffer_rsrc(a.sx + t.r, static_cast<uint32_t>(t.cols) * 4);
#pragma unroll
        for (int p = 0; p < (PA + PB) / 64; ++p) {
            if (p % W != wave) continue;
            if (p < PA / 64) {
                load_word_to_lds(wr_, (p * 64 + lane) * 4, to + p * 256);
            } else {
                const int n = (p - PA / 64) * 64 + lane;
                uint32_t off = n * 4;
                if (gather) off = n < t.cols && index[n] < static_cast<uint32_t>(a.x_rows) ? index[n] * 4 : kPastEnd;
                load_word_to_lds(xr, off, to + p * 256);
            }
        }
    }
    // Start stage s's loads.  Chunks past the last, and everything behind the last
    // item, are zeros.
    __device__ __forceinline__ void issue(int s, int slot, bool there) const {
        const uint32_t to = lds0 + slot * Stage + wave * 1024;
        const int chunks = there ? a.chunks : 0;
        const auto row_loads = [&](auto nt) {
#pragma unroll
            for (int i = 0; i < ALoads; ++i) {
                const int c = i * W + wave, tile = c % ATiles, k = s * KS + c / ATiles;
                const uint32_t off = k < chunks ? aoff + ((tile >> 2) * a.chunks + k) * kI8BlockBytes + (tile & 3) * 1024 : kPastEnd;
                if constexpr (nt) load_to_lds_nt(ar, off, to + i * W * 1024);
                else load_to_lds(ar, off, to + i * W * 1024);
            }
        };
        if (once) row_loads(std::true_type{});
        else row_loads(std::false_type{});
#pragma unroll
        for (int i = 0; i < BLoads; ++i)
            load_to_lds(br, s * KS + load_chunk(i) < chunks ? boff[i] + s * (KS * kI8Chunk) : kPastEnd, to + ABytes + i * W * 1024);
    }
    struct Frags {
        uint4 w[TM], x[TN];
    };
    __device__ __forceinline__ void read(int slot, int chunk, Frags &f) const {
        const uint8_t *p = lds + slot * Stage;
#pragma unroll
        for (int t = 0; t < TN; ++t)
            f.x[t] = *reinterpret_cast<const uint4 *>(p + ABytes + (chunk * BTiles + wc * TN + t) * 1024 + bread);
#pragma unroll
        for (int i = 0; i < TM; ++i)
            f.w[i] = *reinterpret_cast<const uint4 *>(p + (chunk * ATiles + wr * TM + i) * 1024 + lane * 16);
    }
    __device__ __forceinline__ static void multiply(const Frags &f, i32x4 (&acc)[TM][TN]) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < TN; ++t) acc[i][t] = i8_dot(f.w[i], f.x[t], acc[i][t]);
    }
    __device__ __forceinline__ static void barrier() {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    // An item every result of which is stored: `Stores` instructions of a wave at least,
    // 16 bytes a lane each.
    static constexpr int Stores = TM * TN * (Form == kStoreMiddle ? 8 : Bytes * 4) / 16;
    __device__ __forceinline__ bool whole(const I8Item &t) const {
        return t.cols == BN && (Form == kStoreMiddle ? (t.m0 + BM + 127) / 128 * 64 : t.m0 + BM) <= a.M;
    }
    // All items first, first + step, .. below end; item(i) says which that is.
    template<class Fetch, class Store>
    __device__ __forceinline__ void run(int first, int step, int end, const Fetch &fetch, const Store &store) {
        if (first >= end) return;
        // Two chunks a turn of the loop below: an odd last one has a partner of zeros.
        const int stages = KS == 1 ? (a.chunks + 1) / 2 * 2 : (a.chunks + KS - 1) / KS;
        // The loading side: item `at`, the `number`-th here, its next stage, and the item after it.
        int at = first, number = 0, stage = 0;
        I8Item next = fetch(first);
        load_index(next, 0);
        wait_for_lds_loads<0>();
        const auto begin = [&](bool arrived) {
            if (!arrived) wait_for_lds_loads<0>();
            start(next, number);
            if (at + step < end) {
                next = fetch(at + step);
                load_index(next, number + 1);
            }
        };
        begin(true);
        const auto advance = [&](int slot, bool arrived) {
            issue(stage, slot, at < end);
            if (at < end && ++stage == stages) {
                stage = 0;
                at += step;
                ++number;
                if (at < end) begin(arrived);
            }
        };
#pragma unroll
        for (int s = 0; s < S - 1; ++s) advance(s, false);
        wait_for_lds_loads<(S - 2) * Loads>();
        barrier();
        Frags f[2];
        read(0, 0, f[0]);
        int slot = 0;   // of the current stage
        // The next stage is there, for every wave, and the last one's buffer, which no
        // wave reads any more, takes the stage S - 1 ahead.  An item's indices were
        // on their way `stages` turns before it begins, and what was S - 2 turns ago
        // has arrived.
        // A wave's memory operations complete in the order in which it issued them, so
        // that for S - 2 turns the last item's stores, issued behind the loads waited
        // for, may still be on their way (163,840 rows of 512 x 2048 matrices 373 -> 369 us).
        int stored = 0;   // such turns left
        const auto turn = [&](Frags &into) {
            if (stored > 0) {
                --stored;
                wait_for_lds_loads<(S - 3) * Loads + Stores>();
            } else {
                wait_for_lds_loads<(S - 3) * Loads>();
            }
            barrier();
            advance(slot == 0 ? S - 1 : slot - 1, stages >= S - 2);
            slot = slot + 1 == S ? 0 : slot + 1;
            read(slot, 0, into);
        };
        int done = 0;
        for (int i = first; i < end; i += step, ++done) {
            i32x4 acc[TM][TN];
#pragma unroll
            for (int p = 0; p < TM; ++p)
#pragma unroll
                for (int t = 0; t < TN; ++t) acc[p][t] = i32x4{0, 0, 0, 0};
            if constexpr (KS == 1) {
                for (int s = 0; s < stages; s += 2) {
                    turn(f[1]);
                    multiply(f[0], acc);
                    turn(f[0]);
                    multiply(f[1], acc);
                }
            } else {
                static_assert(KS % 2 == 0);
                for (int s = 0; s < stages; ++s) {
#pragma unroll
                    for (int c = 0; c < KS; ++c) {
                        if (c + 1 < KS) read(slot, c + 1, f[(c + 1) & 1]);
                        else turn(f[(c + 1) & 1]);
                        multiply(f[c & 1], acc);
                    }
                }
            }
            const I8Item item = fetch(i);
            store(item, reinterpret_cast<const float *>(lds + params_at(done)), acc);
            if (whole(item)) stored = S - 2;
        }
        wait_for_lds_loads<0>();   // no load may outlive the buffers
    }

    __device__ __forceinline__ void store_each(size_t at, int m, const float *v, int count) const {
#pragma unroll
        for (int i = 0; i < count; ++i)
            if (m + i < a.M) store1<Y>(a.y, at + i, v[i]);
    }
    __device__ __forceinline__ void store_rows(const I8Item &it, const float *params, const i32x4 (&acc)[TM][TN]) const {
        constexpr int G = TM < 2 ? 1 : 2, R = 4 * G;   // tiles of a run, its length
        const int g = lane >> 4;
#pragma unroll
        for (int p = 0; p < TM; p += G) {
            const int tile = wr * TM + p, first = (tile >> 1) * 32, m = first + g * 8 + (tile & 1) * 4;
            const bool inside = it.m0 + first + 32 <= a.M;
            float sw[R];
#pragma unroll
            for (int i = 0; i < R; ++i) sw[i] = params[m + i];
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int n = (wc * TN + t) * 16 + (lane & 15);
                if (n >= it.cols) continue;
                const float sx = params[PA + n];
                float v[R];
#pragma unroll
                for (int i = 0; i < R; ++i) v[i] = static_cast<float>(acc[p + i / 4][t][i % 4]) * (sx * sw[i]);
                const size_t row = (static_cast<size_t>(it.r) + n) * static_cast<size_t>(a.y_stride) + it.m0;
                if (!inside) {
                    store_each(row + m, it.m0 + m, v, R);
                } else if constexpr (G == 1) {
                    store4<Y>(a.y, row + m, v);
                } else if constexpr (Y == kF32) {
                    // Half of a run for half of the partner's, 32 lanes away, of the same
                    // row: 64 bytes of it a store here as well.
                    float lo[4], hi[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[4 + i]), false, false);
                        lo[i] = __uint_as_float(s[0]);
                        hi[i] = __uint_as_float(s[1]);
                    }
                    const size_t at = row + first + (g & 1) * 8 + (g >> 1) * 4;
                    store4<kF32>(a.y, at, lo);
                    store4<kF32>(a.y, at + 16, hi);
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = Y == kBF16 ? pack_bf16(v[2 * i], v[2 * i + 1]) : pack_f16(v[2 * i], v[2 * i + 1]);
                    __builtin_memcpy(static_cast<uint16_t *>(a.y) + row + m, w, 16);
                }
            }
        }
    }
    // SiLU(gate) * up of pairs of tiles, [rows][I] in fp32.
    __device__ __forceinline__ void store_middle(const I8Item &it, const float *params, const i32x4 (&acc)[TM][TN]) {
        static_assert(Form != kStoreMiddle || TM % 2 == 0);
#pragma unroll
        for (int p = 0; p < TM; p += 2) {
            const int tile = it.m0 / 16 + wr * TM + p, in = (tile & 7) * 8 + (lane >> 4) * 4, at = (tile >> 3) * 64 + in;   // tile is even
            if (at >= a.M) continue;
            const float *s = params + ((tile >> 3) - it.m0 / 128) * 128 + in;
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int n = (wc * TN + t) * 16 + (lane & 15);
                if (n >= it.cols) continue;
                const float sx = params[PA + n];
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    v[q] = silu_product(static_cast<float>(acc[p][t][q]) * (sx * s[q]),
                                        static_cast<float>(acc[p + 1][t][q]) * (sx * s[64 + q]), flags);
                store4<kF32>(a.y, (static_cast<size_t>(it.r) + n) * static_cast<size_t>(a.y_stride) + at, v);
            }
        }
    }
};

}  // namespace
}  // namespace moe
