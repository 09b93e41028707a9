// The 8-bit integer operators: int8 matrices with one fp32 scale per output
// channel, int8 activations with one per row.  gfx950 (CDNA4), wave64.
//   y[n][m] = (sum_k cx[n][k] cw[m][k]) * (sx[n] * sw[m])
// The sum is a whole number that int32 holds (2^28 at most: K <= 16384), so its
// order, the tile and the number of waves that share K change no bit of y.
//
// Matrix layout.  A matrix [M][K] is kept as tiles of 16 rows x 64 columns (1
// KiB, zero past its edges), [ceil(M/16)][ceil(K/64)], in the order in which a
// wave's lanes take them as an operand of v_mfma_i32_16x16x64_i8: lane l holds
// row l % 16, columns 16 (l / 16) .. + 15.  A tile is one contiguous KiB, from
// HBM or from LDS.  What a product reads past a row of activations meets the
// zeros past the matrix row, so rows need no padding.
#pragma once

#include "moe_fp8.hpp"   // element types, loads into LDS

namespace moe {

inline constexpr int kI8TileRows = 16, kI8Chunk = 64, kI8TileBytes = kI8TileRows * kI8Chunk;
__host__ __device__ constexpr int i8_chunks(int cols) { return (cols + kI8Chunk - 1) / kI8Chunk; }

// Canonical int8 codes [matrices][rows][cols] -> tiles.  pairs: tile i becomes tile
// 2 i + shift, so that gate (shift 0) and up rows (shift 1) alternate in tiles of
// 16; rows is then a multiple of 16.
hipError_t launch_i8_repack(const int8_t *codes, uint8_t *tiles, size_t matrices, int rows, int cols, bool pairs, int shift,
                            hipStream_t s);
// Rows of `type` -> codes [rows][pitch], scales [rows].
hipError_t launch_quantize_i8(const void *x, int type, int64_t stride, int width, size_t rows, int8_t *codes, int64_t pitch,
                              float *scales, int *error, hipStream_t s);

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
__device__ __forceinline__ uint2 quantize8_i8(const float (&v)[8], const GroupScale &s) {
    if (s.bad) return make_uint2(0u, 0u);
    return make_uint2(pack_i8(v[0] * s.r, v[1] * s.r, v[2] * s.r, v[3] * s.r),
                      pack_i8(v[4] * s.r, v[5] * s.r, v[6] * s.r, v[7] * s.r));
}

// One tile's products onto acc: lane l has rows 4 (l / 16) + i of the tile against
// token l % 16.
__device__ __forceinline__ i32x4 i8_dot(const uint4 &w, const uint4 &x, const i32x4 &acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), acc, 0, 0, 0);
}

// What a product writes: rows of y, or SiLU(gate) * up in fp32 from matrices whose
// gate and up rows alternate in tiles of 16.
enum { kStoreRows = 0, kStoreMiddle = 1 };

struct I8Args {
    const uint8_t *tiles;     // [experts][ceil(M/16)][chunks] tiles
    const float *sw;          // [experts][M], in the tiles' order of rows
    const int8_t *x;          // rows [..][pitch]
    const float *sx;
    int64_t pitch;
    const int32_t *index;     // row of x of each row of the product, or null: the same
    int x_rows;               // rows of x
    const int32_t *offsets;   // [experts + 1]: rows of each expert's matrix; null: one matrix takes all rows
    int experts;
    void *y;                  // rows of y_type, y_stride apart; kStoreMiddle: fp32
    int64_t y_stride;
    int M, N, K, chunks;      // matrix rows, rows of the product
    int tiles_m;
    int *error;
};

// A workgroup of WR x WC waves takes 16 TM WR rows of the matrix and 16 TN WC
// rows of x, and steps through K in stages of KS chunks, the next stages' operands
// on the way to a ring of S buffers in LDS and the next chunk's from there to
// registers.  A barrier a stage, with the products of the stage's last chunk still
// to be issued behind it: their operands are in registers, so the barrier and the
// LDS reads after it cost the matrix cores nothing.
template<int WR, int WC, int TM, int TN, int S, int KS>
struct I8Tile {
    static constexpr int W = WR * WC, BM = 16 * TM * WR, BN = 16 * TN * WC;
    static constexpr int ATiles = BM / 16, BTiles = BN / 16;
    static constexpr int ABytes = ATiles * KS * kI8TileBytes, Stage = ABytes + BTiles * KS * kI8TileBytes;
    static constexpr int ALoads = ATiles * KS / W, BLoads = BTiles * KS / W, Loads = ALoads + BLoads;   // of a wave and stage
    static constexpr int Pitch = BM * 2 + 8;   // 16-bit results on their way along the rows
    static constexpr int Lds = S * Stage > BN * Pitch ? S * Stage : BN * Pitch;
    static_assert(S >= 3 && ATiles * KS % W == 0 && BTiles * KS % W == 0, "every wave issues the same loads");
    static constexpr uint32_t kPastEnd = 0xc0000000u;   // past every resource here, and no sum with it wraps

    int lane, wave, wr, wc, chunks;
    uint32_t lds0, bread;
    __amdgpu_buffer_rsrc_t ar, br;
    uint32_t aoff[ALoads], boff[BLoads];
    int achunk[ALoads], bchunk[BLoads];

    __device__ __forceinline__ explicit I8Tile(const void *lds) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wr = wave / WC;
        wc = wave % WC;
        lds0 = lds_offset(lds);
        // Fragment of row l % 16, piece l / 16, in the permuted order.
        bread = (lane & 15) * 64 + ((lane >> 4) ^ (lane >> 1 & 3)) * 16;
    }
    // Rows m0 .. of expert e's matrix, rows n0 .. n0 + cols - 1 of the product.
    __device__ __forceinline__ void start(const I8Args &a, int e, int m0, size_t n0, int cols, int &flags) {
        chunks = a.chunks;
        const int row_tiles = (a.M + 15) / 16;
        const uint32_t tile_row = static_cast<uint32_t>(a.chunks) * kI8TileBytes;   // bytes of 16 rows
        ar = buffer_rsrc(a.tiles + (static_cast<size_t>(e) * row_tiles + m0 / 16) * tile_row,
                         static_cast<uint32_t>(min(row_tiles - m0 / 16, ATiles)) * tile_row);
#pragma unroll
        for (int i = 0; i < ALoads; ++i) {
            const int c = i * W + wave;
            achunk[i] = c / ATiles;
            aoff[i] = (c % ATiles) * tile_row + achunk[i] * kI8TileBytes + lane * 16;
        }
        const int8_t *base = a.x;
        if (a.index) {
            br = buffer_rsrc(base, static_cast<uint32_t>((static_cast<size_t>(a.x_rows) - 1) * a.pitch + a.K));
        } else {
            base += n0 * a.pitch;
            br = buffer_rsrc(base, static_cast<uint32_t>(static_cast<size_t>(cols - 1) * a.pitch + a.K));
        }
        // 16 rows of 64 bytes a load, each row's four pieces permuted by its index
        // so that the fragment reads spread over the LDS banks.
        const int r = lane >> 2, piece = (lane & 3) ^ (r >> 1 & 3);
#pragma unroll
        for (int i = 0; i < BLoads; ++i) {
            const int c = i * W + wave, n = c % BTiles * 16 + r;
            bchunk[i] = c / BTiles;
            uint32_t off = kPastEnd;   // rows past the end are read as zeros
            if (n < cols) {
                uint32_t row = static_cast<uint32_t>(n);
                if (a.index) {
                    row = static_cast<uint32_t>(a.index[n0 + n]);
                    if (row >= static_cast<uint32_t>(a.x_rows)) flags |= 1;
                }
                if (!a.index || row < static_cast<uint32_t>(a.x_rows))
                    off = row * static_cast<uint32_t>(a.pitch) + bchunk[i] * kI8Chunk + piece * 16;
            }
            boff[i] = off;
        }
    }
    // Start stage s's loads.  Chunks past the last are zeros.
    __device__ __forceinline__ void issue(int s, int slot) const {
        const uint32_t to = lds0 + slot * Stage + wave * 1024;
#pragma unroll
        for (int i = 0; i < ALoads; ++i)
            load_to_lds(ar, s * KS + achunk[i] < chunks ? aoff[i] + s * (KS * kI8TileBytes) : kPastEnd, to + i * W * 1024);
#pragma unroll
        for (int i = 0; i < BLoads; ++i)
            load_to_lds(br, s * KS + bchunk[i] < chunks ? boff[i] + s * (KS * kI8Chunk) : kPastEnd,
                        to + ABytes + i * W * 1024);
    }
    struct Frags {
        uint4 w[TM], x[TN];
    };
    __device__ __forceinline__ void read(const uint8_t *lds, int slot, int chunk, Frags &f) const {
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
    __device__ __forceinline__ void product(const uint8_t *lds, i32x4 (&acc)[TM][TN]) const {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < TN; ++t) acc[i][t] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S - 1; ++s) issue(s, s);
        wait_for_lds_loads<(S - 2) * Loads>();
        barrier();
        Frags f[2];
        read(lds, 0, 0, f[0]);
        const int stages = (chunks + KS - 1) / KS;
        int slot = 0;   // of the current stage
        // Stage s's last chunk: stage s + 1 is there, for every wave, and s - 1's
        // buffer, which no wave reads any more, takes stage s + S - 1.
        const auto turn = [&](int s, Frags &next) {
            wait_for_lds_loads<(S - 3) * Loads>();
            barrier();
            issue(s + S - 1, slot == 0 ? S - 1 : slot - 1);
            slot = slot + 1 == S ? 0 : slot + 1;
            read(lds, slot, 0, next);
        };
        if constexpr (KS == 1) {
            int s = 0;
            for (; s + 1 < stages; s += 2) {
                turn(s, f[1]);
                multiply(f[0], acc);
                turn(s + 1, f[0]);
                multiply(f[1], acc);
            }
            if (s < stages) multiply(f[0], acc);
        } else {
            static_assert(KS % 2 == 0);
            for (int s = 0; s < stages; ++s) {
#pragma unroll
                for (int c = 0; c < KS; ++c) {
                    if (c + 1 < KS) read(lds, slot, c + 1, f[(c + 1) & 1]);
                    else turn(s, f[(c + 1) & 1]);
                    multiply(f[c & 1], acc);
                }
            }
        }
        wait_for_lds_loads<0>();   // no load may outlive the buffers
        __syncthreads();
    }

    // Scale of row n0 + n of the product; 0 past the end and for a row that is not there.
    __device__ __forceinline__ static float row_factor(const I8Args &a, size_t n0, int n, int cols) {
        if (n >= cols) return 0.0f;
        if (!a.index) return a.sx[n0 + n];
        const uint32_t row = static_cast<uint32_t>(a.index[n0 + n]);
        return row < static_cast<uint32_t>(a.x_rows) ? a.sx[row] : 0.0f;
    }
    // Rows m .. m + 3's scales.
    __device__ __forceinline__ static void channel_factors(const I8Args &a, int e, int m, float (&f)[4]) {
        const float *p = a.sw + static_cast<size_t>(e) * a.M;
#pragma unroll
        for (int q = 0; q < 4; ++q) f[q] = p[min(m + q, a.M - 1)];
    }
    // 16-bit results by way of LDS, so that a wave's stores run along the rows of
    // y; fp32 ones, twice as long, straight from the sums.
    template<int Y>
    __device__ __forceinline__ void store_rows(const I8Args &a, int e, int m0, size_t n0, int cols, const i32x4 (&acc)[TM][TN],
                                               uint8_t *lds) const {
        float sx[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) sx[t] = row_factor(a, n0, (wc * TN + t) * 16 + (lane & 15), cols);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = (wr * TM + i) * 16 + (lane >> 4) * 4;
            float sw[4];
            channel_factors(a, e, m0 + m, sw);
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int n = (wc * TN + t) * 16 + (lane & 15);
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = static_cast<float>(acc[i][t][q]) * (sx[t] * sw[q]);
                if constexpr (Y != kF32) {
                    store4<Y>(lds + n * Pitch, m, v);
                } else if (n < cols) {
                    const size_t at = (n0 + n) * static_cast<size_t>(a.y_stride) + m0 + m;
                    if (m0 + m + 3 < a.M) {
                        store4<Y>(a.y, at, v);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (m0 + m + q < a.M) store1<Y>(a.y, at + q, v[q]);
                    }
                }
            }
        }
        if constexpr (Y != kF32) {
            constexpr int Lanes = BM / 4;   // lanes of a row
            static_assert(64 * W % Lanes == 0);
            __syncthreads();
            const int c = static_cast<int>(threadIdx.x) % Lanes * 4;
#pragma unroll 4
            for (int n = static_cast<int>(threadIdx.x) / Lanes; n < cols; n += 64 * W / Lanes) {
                uint2 w;
                __builtin_memcpy(&w, lds + n * Pitch + c * 2, 8);
                uint16_t *y = static_cast<uint16_t *>(a.y) + (n0 + n) * static_cast<size_t>(a.y_stride) + m0 + c;
                if (m0 + c + 3 < a.M) {
                    __builtin_memcpy(y, &w, 8);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (m0 + c + q < a.M) y[q] = static_cast<uint16_t>((q < 2 ? w.x : w.y) >> (16 * (q & 1)));
                }
            }
        }
    }
    // SiLU(gate) * up of the pairs of row tiles; every row of the matrix is there
    // (its rows are a multiple of 64).
    __device__ __forceinline__ void store_middle(const I8Args &a, int e, int m0, size_t n0, int cols,
                                                 const i32x4 (&acc)[TM][TN], int &flags) const {
        static_assert(TM % 2 == 0);
        float sx[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) sx[t] = row_factor(a, n0, (wc * TN + t) * 16 + (lane & 15), cols);
#pragma unroll
        for (int i = 0; i < TM; i += 2) {
            const int m = m0 + (wr * TM + i) * 16 + (lane >> 4) * 4, j = m / 32 * 16 + m % 16;
            if (m >= a.M) continue;
            float sg[4], su[4];
            channel_factors(a, e, m, sg);
            channel_factors(a, e, m + 16, su);
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                const int n = (wc * TN + t) * 16 + (lane & 15);
                if (n >= cols) continue;
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    v[q] = silu_mul(static_cast<float>(acc[i][t][q]) * (sx[t] * sg[q]),
                                    static_cast<float>(acc[i + 1][t][q]) * (sx[t] * su[q]), flags);
                store4<kF32>(a.y, (n0 + n) * static_cast<size_t>(a.y_stride) + j, v);
            }
        }
    }
};

}  // namespace
}  // namespace moe
