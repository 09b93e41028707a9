// The 8-bit floating point operators: e4m3 values (OCP: 4 exponent bits of
// bias 7, 3 mantissa bits, no infinities, at most 448) with one fp32 scale
// per block, 128 consecutive elements of an activation row or 128 x 128
// elements of a matrix.  gfx950 (CDNA4), wave64.
//
// Matrix layout.  A matrix [M][K] is kept as tiles of 16 rows x 128 columns
// (2 KiB, zero past its edges), [ceil(M/16)][ceil(K/128)], in the order in
// which a wave's lanes take them as an MFMA operand: lane l holds row l % 16,
// columns 32 (l / 16) .. + 31, as two 16-byte chunks; the tile is [chunk][lane]
// [16 B].  One tile is one K step of v_mfma_f32_16x16x128_f8f6f4 and one scale
// block, a wave reads it as two contiguous KiB, from HBM or from LDS, and rows
// stream through memory in the order they are used.  An MFMA sums over its K
// whatever order both operands share, so the same 32 bytes are also four steps
// of v_mfma_f32_16x16x32_f16 (step s: bytes 8 s .. + 7 of every lane).
#pragma once

#include "moe_device.hpp"

namespace moe {

inline constexpr int kFp8Block = 128;       // elements per scale along a row; rows per scale of a matrix
inline constexpr int kFp8TileRows = 16;
inline constexpr int kFp8TileBytes = kFp8TileRows * kFp8Block;
// Element types of the entry points (MOE_F32, MOE_BF16, MOE_F16).
inline constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;
__host__ __device__ constexpr int elem_bytes(int type) { return type == kF32 ? 4 : 2; }
// Sources of e4m3 columns that are quantised before a product: rows and tiles.
inline constexpr int kCodes = 3, kTiles = 4;

// Canonical e4m3 codes [rows][cols] -> tiles.  cols % 16 == 0.
hipError_t launch_fp8_repack(const uint8_t *codes, uint8_t *tiles, size_t rows, int cols, hipStream_t s);
// Rows of `type` -> codes [columns][width] and scales [columns][ceil(width/128)].
hipError_t launch_quantize_e4m3(const void *x, int type, int64_t stride, int width, int columns, uint8_t *codes,
                                float *scales, int *error, hipStream_t s);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// --------------------------------------------------------- element types ---
template<int T>
__device__ __forceinline__ float load1(const void *p, size_t i) {
    if constexpr (T == kF32) return static_cast<const float *>(p)[i];
    else if constexpr (T == kBF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t *>(p)[i]) << 16);
    else return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
}
template<int T>
__device__ __forceinline__ void store1(void *p, size_t i, float v) {
    if constexpr (T == kF32) static_cast<float *>(p)[i] = v;
    else if constexpr (T == kBF16) static_cast<__bf16 *>(p)[i] = static_cast<__bf16>(v);
    else static_cast<_Float16 *>(p)[i] = static_cast<_Float16>(v);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
// Eight consecutive elements as they lie in memory: 16-bit types fill lo.
struct Raw8 {
    uint4 lo, hi;
};
template<int T>
__device__ __forceinline__ Raw8 load8_raw(const void *p, size_t i) {
    Raw8 r;
    if constexpr (T == kF32) {
        const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + i);
        r.lo = q[0];
        r.hi = q[1];
    } else {
        r.lo = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
        r.hi = r.lo;
    }
    return r;
}
template<int T>
__device__ __forceinline__ void unpack8(const Raw8 &r, float (&v)[8]) {
    const uint32_t lo[4] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w}, hi[4] = {r.hi.x, r.hi.y, r.hi.z, r.hi.w};
    if constexpr (T == kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(lo[i]); v[4 + i] = __uint_as_float(hi[i]); }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kBF16) {
                v[2 * i] = __uint_as_float(lo[i] << 16);
                v[2 * i + 1] = __uint_as_float(lo[i] & 0xffff0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, lo[i]);
                v[2 * i] = static_cast<float>(h[0]);
                v[2 * i + 1] = static_cast<float>(h[1]);
            }
        }
    }
}
// Eight elements at any alignment of their type (the hardware takes such 16-byte
// accesses), of which the first `valid` are the row's; 0 after those.
template<int T>
__device__ __forceinline__ Raw8 load8_any(const void *p, size_t at, int valid) {
    Raw8 r{};
    const char *q = static_cast<const char *>(p) + at * elem_bytes(T);
    if (valid >= 8) {
        __builtin_memcpy(&r.lo, q, 16);
        if constexpr (T == kF32) __builtin_memcpy(&r.hi, q + 16, 16);
    } else if (valid > 0) {
        uint32_t w[8] = {};
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            if (i >= valid) break;
            if constexpr (T == kF32) w[i] = reinterpret_cast<const uint32_t *>(q)[i];
            else w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(q)[i]) << (16 * (i & 1));
        }
        r.lo = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (T == kF32) r.hi = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return r;
}
// Four consecutive results, 16 or 8 bytes at any alignment of their type (the
// hardware takes such stores).
template<int T>
__device__ __forceinline__ void store4(void *p, size_t i, const float (&v)[4]) {
    char *q = static_cast<char *>(p) + i * elem_bytes(T);
    if constexpr (T == kF32) {
        __builtin_memcpy(q, v, 16);
    } else {
        const uint2 w = T == kBF16 ? make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]))
                                   : make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]));
        __builtin_memcpy(q, &w, 8);
    }
}

// ---------------------------------------------------------- quantisation ---
// The scale of a group whose largest magnitude has the bits `amax`:
//   a = max(|x|max, 2^-100), s = a / 448, r = 448 / a (both correctly rounded)
// and the codes are e4m3(x * r), to nearest even.  The floor keeps r finite;
// what lies below its half step becomes 0.  Integer order of the magnitudes'
// bits is their order as numbers, with infinities and NaN above all: `bad`
// marks a group that holds one, whose codes and scale are then all zero.
struct GroupScale {
    float s, r;
    bool bad;
};
__device__ __forceinline__ GroupScale group_scale(uint32_t amax) {
    const bool bad = amax >= 0x7f800000u;
    const float a = fmaxf(__uint_as_float(bad ? 0u : amax), 0x1p-100f);
    return GroupScale{bad ? 0.0f : a / 448.0f, 448.0f / a, bad};
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// e4m3 codes of four values.  |v| <= 448 (1 + 2^-23): below 464, from where
// the conversion gives NaN instead of 448.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return static_cast<uint32_t>(w);
}

// The largest magnitude of 16 neighbouring lanes' eight values.
__device__ __forceinline__ uint32_t max16(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
    m = max(m, static_cast<uint32_t>(lane_xor<1>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<2>(static_cast<int>(m))));
    m = max(m, static_cast<uint32_t>(lane_xor<4>(static_cast<int>(m))));
    return max(m, static_cast<uint32_t>(lane_xor<8>(static_cast<int>(m))));
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], const GroupScale &s) {
    if (s.bad) return make_uint2(0u, 0u);
    return make_uint2(pack_e4m3(v[0] * s.r, v[1] * s.r, v[2] * s.r, v[3] * s.r),
                      pack_e4m3(v[4] * s.r, v[5] * s.r, v[6] * s.r, v[7] * s.r));
}
// Where a tile holds elements 8 part .. + 7 of a row's block.
__device__ __forceinline__ int tile_offset(int part, int row) {
    return ((part >> 1) & 1) * 1024 + ((part >> 2) * 16 + row) * 16 + (part & 1) * 8;
}

// ---------------------------------------------------------------- products ---
// Eight e4m3 codes as fp16, which holds every e4m3 value exactly (NaN too).
__device__ __forceinline__ f16x8 e4m3_to_f16(uint32_t lo, uint32_t hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// A lane's 32 codes of one tile (or of one token's block).
struct Frag {
    uint4 c0, c1;
};
struct FragF16 {
    f16x8 s[4];
};
__device__ __forceinline__ FragF16 to_f16(const Frag &f) {
    return FragF16{{e4m3_to_f16(f.c0.x, f.c0.y), e4m3_to_f16(f.c0.z, f.c0.w), e4m3_to_f16(f.c1.x, f.c1.y),
                    e4m3_to_f16(f.c1.z, f.c1.w)}};
}
// A fragment as the operand of block_dot.
template<class Operand>
__device__ __forceinline__ Operand operand(const Frag &f) {
    if constexpr (sizeof(Operand) == sizeof(Frag)) return f;
    else return to_f16(f);
}
// One block's products summed from zero: lane l gets rows 4 (l / 16) + i of
// the tile against token l % 16.
//
// On fp16 operands the sums are fp32 sums (2-norm of the error 1e-8 of the
// result's on normal data).  The e4m3 MFMA has twice the rate, but cuts bits: of
// the products of eight codes next to each other, 8 i .. + 7, with 2^e the
// largest product of two codes' powers of two (2^-6 for a subnormal code), it
// keeps each down to 2^(e - 13), rounded toward zero; the sum of the eight is
// exact, and sums are added in fp32.  So a product loses bits where another of
// its eight is about 2^7 times as large, and less than 2^-13 of that one (2^-10
// where it has a subnormal code).  2-norm of the error: 1.5e-5 of the result's
// on normal data, 5.5e-5 with an element of each group of 128 two hundred times
// the others' deviation, 5e-5 on codes drawn evenly.  Fit for results that are
// rounded to 16 bits (by up to 2^-8 or 2^-11 of themselves), where the caller has
// not asked for fp32 sums, not for fp32 ones.
__device__ __forceinline__ f32x4 block_dot(const FragF16 &w, const FragF16 &x) {
    f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.s[s], x.s[s], p, 0, 0, 0);
    return p;
}
__device__ __forceinline__ f32x4 block_dot(const Frag &w, const Frag &x) {
    const f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(i32x8, w), __builtin_bit_cast(i32x8, x), z,
                                                            0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ Frag load_tile(const uint8_t *tile, int lane) {
    const uint4 *p = reinterpret_cast<const uint4 *>(tile) + lane;
    return Frag{p[0], p[64]};
}

// 16 bytes a lane from memory (base r, byte offset off, zero past r's end)
// straight into LDS, lane i's at byte 16 i from `lds`, which is the same for
// the whole wave.  Written in assembly, without output registers: the compiler
// orders every LDS read behind such a load that it knows of, where here only
// the wait and the barrier before a buffer's first read have to.  Nothing but
// those may read what it writes.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
// The same with 4 bytes a lane.
__device__ __forceinline__ void load_word_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :: "s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
// Until at most N of the wave's loads are outstanding.
template<int N>
__device__ __forceinline__ void wait_for_lds_loads() {
    static_assert(N < 64);
    asm volatile("s_waitcnt vmcnt(%0)" :: "i"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_offset(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void *)p));
}

}  // namespace
}  // namespace moe
