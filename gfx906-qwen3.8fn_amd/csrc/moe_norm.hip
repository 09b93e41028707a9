// The norms after one block and before the next with the gate, the scales and
// the residual sum between them (moe_block_norm), one pass over the rows:
//   b = post_weight ? rms(block) (offset + post_weight) : block
//   h = residual_scale residual + block_scale gate b
//   n = rms(h) (offset + pre_weight),   rms(v) = v / sqrt(mean(v^2) + eps)
// n may be written as values, as Q8_1 rows and as e4m3 rows at once: the
// router reads values and the experts' products read quantised rows.
#include "moe_ffn.h"
#include "moe_fp8.hpp"

#include <algorithm>

namespace moe {
namespace {

// Waves a CU of a long batch (16,384 rows, us at 16 / 24 / 32: 2,560 bf16
// channels with an element gate 88 / 101 / 112, 2,048 fp32 ones 104 / 106 / 103).
inline constexpr int kNormWaves = 16;

struct NormArgs {
    const void *residual, *block, *gate;
    void *residual_out, *out;
    int64_t residual_stride, block_stride, gate_stride, residual_out_stride, out_stride;
    const float *post_weight, *pre_weight;
    uint32_t *q8;
    uint8_t *codes;
    float *scales;
    int *error;
    float eps, offset, residual_scale, block_scale;
    int hidden, tokens, gate_form, gate_sigmoid;
};

// The counterpart of load8_any.
template<int T>
__device__ __forceinline__ void store8_any(void *p, size_t at, int valid, const float (&v)[8]) {
    char *q = static_cast<char *>(p) + at * elem_bytes(T);
    if (valid >= 8) {
        if constexpr (T == kF32) {
            __builtin_memcpy(q, v, 32);
        } else {
            const auto pack = [](float a, float b) { return T == kBF16 ? pack_bf16(a, b) : pack_f16(a, b); };
            const uint4 w = make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
            __builtin_memcpy(q, &w, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < valid) store1<T>(q, i, v[i]);
    }
}

// The sum over the workgroup, by a butterfly in each wave and then in wave
// order.  Consecutive sums alternate between two slots: a wave writes a slot
// again only after the barrier of the sum between, which no wave reaches
// before it has read the slot.
__device__ __forceinline__ float group_sum(float v, float (*slot)[16], int &which) {
    v = xor_sum_from<32>(v);
    const int W = blockDim.x >> 6;
    if (W == 1) return v;
    which ^= 1;
    if ((threadIdx.x & 63) == 0) slot[which][threadIdx.x >> 6] = v;
    __syncthreads();
    float s = slot[which][0];
    for (int w = 1; w < W; ++w) s = s + slot[which][w];
    return s;
}

// A Q8_1 block from four neighbouring lanes with 8 elements each: the bytes
// and flags of moe_quantize_q8_1 for the same fp32 row (its pairwise sum is a
// subtree of the raw sum's XOR butterfly in every lane, combined in order).
__device__ __forceinline__ void store_q8(uint32_t *q8, size_t block, int part, float (&v)[8], bool in, int &flags) {
    int bad = 0;
    float amax = 0.0f, t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!isfinite(v[i])) { bad = 1; v[i] = 0.0f; }
        amax = fmaxf(amax, fabsf(v[i]));
        t[i] = v[i];
    }
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) t[i] = t[2 * i] + t[2 * i + 1];
    amax = fmaxf(amax, lane_xor<1>(amax));
    amax = fmaxf(amax, lane_xor<2>(amax));
    bad |= lane_xor<1>(bad);
    bad |= lane_xor<2>(bad);
    const float sum = xor_sum<2>(xor_sum<1>(t[0])), d = amax / 127.0f;
    const uint32_t hd = f2h(d), hs = f2h(sum);
    const bool representable = isfinite(sum) && (hs & 0x7c00u) != 0x7c00u && (hd & 0x7c00u) != 0x7c00u &&
                               (amax == 0.0f || d > 0.0f);
    const bool quant = !bad && representable && amax != 0.0f;
    uint32_t words[2];
    int bad_code = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        words[w] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float c = quant ? roundf(v[4 * w + b] / d) : 0.0f;
            bad_code |= !isfinite(c) || c < -127.0f || c > 127.0f;
            words[w] |= (static_cast<uint32_t>(static_cast<int>(c)) & 0xffu) << (8 * b);
        }
    }
    bad_code |= lane_xor<1>(bad_code);
    bad_code |= lane_xor<2>(bad_code);
    const bool valid = !bad && representable && !bad_code;
    if (!in) return;
    uint32_t *out = q8 + block * 9;
    if (part == 0) out[0] = valid && amax != 0.0f ? hd | (hs << 16) : 0u;
    out[1 + 2 * part] = valid ? words[0] : 0u;
    out[2 + 2 * part] = valid ? words[1] : 0u;
    flags |= (bad ? 1 : 0) | ((representable && !bad_code) ? 0 : 2);
}

// An e4m3 group from 16 neighbouring lanes, as k_quantize_e4m3 forms it.
__device__ __forceinline__ void store_e4m3(uint8_t *codes, size_t at, float *scale, int part, const float (&v)[8], int valid,
                                           int &flags) {
    const GroupScale g = group_scale(max16(v));
    const uint2 c = quantize8(v, g);
    if (valid >= 8) {
        __builtin_memcpy(codes + at, &c, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < valid) codes[at + i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
    if (part == 0 && valid > 0) *scale = g.s;
    if (g.bad) flags |= 1;
}

// A workgroup takes rows blockIdx.x, + gridDim.x, .., 8 NV elements a thread
// and all of a row in registers.  Weights and a gate per channel stay in
// registers and a row is on its way while the last one is reduced (NV = 1; with
// 16 elements a thread the registers do not suffice for that, and an element
// gate is read where it is used: 2,000 rows of 16,384 bf16 channels 72 us, 3.6
// TB/s, and 87 with such a gate; 80 and 117 when it was read with the rest.  fp16
// 72 and 88, fp32 120 and 136 us, 4.4 and 4.8 TB/s, though fp16 spills seven
// registers there and fp32 three).
// TB: type of block, out and an element gate; TR: of the residual.
template<int TB, int TR, int NV>
__global__ __launch_bounds__(1024) void k_block_norm(NormArgs a) {
    __shared__ float slots[2][16];
    const int tid = threadIdx.x, H = a.hidden, nb = (H + kFp8Block - 1) / kFp8Block;
    int col[NV], valid[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        col[j] = (j * static_cast<int>(blockDim.x) + tid) * 8;
        valid[j] = min(8, H - col[j]);   // <= 0 past the row's end
    }
    const auto channels = [&](const void *p, int j, float (&w)[8]) { unpack8<kF32>(load8_any<kF32>(p, col[j], valid[j]), w); };
    float post[8], pre[8], gate[8];   // NV = 1
    if constexpr (NV == 1) {
        if (a.post_weight) channels(a.post_weight, 0, post);
        if (a.pre_weight) channels(a.pre_weight, 0, pre);
        if (a.gate_form == MOE_GATE_CHANNEL) {
            channels(a.gate, 0, gate);
            if (a.gate_sigmoid) {
#pragma unroll
                for (int i = 0; i < 8; ++i) gate[i] = sigmoid(gate[i]);
            }
        }
    }
    Raw8 nr[NV], nblk[NV], ng[NV];   // the next row
    float token_gate = 0.0f;
    const auto load = [&](size_t n) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nr[j] = load8_any<TR>(a.residual, n * a.residual_stride + col[j], valid[j]);
            if (a.block) nblk[j] = load8_any<TB>(a.block, n * a.block_stride + col[j], valid[j]);
            if (NV == 1 && a.gate_form == MOE_GATE_ELEMENT) ng[j] = load8_any<TB>(a.gate, n * a.gate_stride + col[j], valid[j]);
        }
        if (a.gate_form == MOE_GATE_TOKEN) token_gate = static_cast<const float *>(a.gate)[n];
    };
    int flags = 0, which = 0;
    if constexpr (NV == 1) load(blockIdx.x);
    for (int n = blockIdx.x; n < a.tokens; n += gridDim.x) {
        float r[NV][8], b[NV][8], g[8];
        if constexpr (NV > 1) load(n);
        float row_gate = token_gate;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack8<TR>(nr[j], r[j]);
            if (a.block) unpack8<TB>(nblk[j], b[j]);
            if (NV == 1 && a.gate_form == MOE_GATE_ELEMENT) unpack8<TB>(ng[j], g);
        }
        if (NV == 1 && n + static_cast<int>(gridDim.x) < a.tokens) load(n + gridDim.x);
        if (a.block) {
            if (a.post_weight) {
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) s = fmaf(b[j][i], b[j][i], s);
                s = group_sum(s, slots, which);
                const float scale = 1.0f / sqrtf(s / static_cast<float>(H) + a.eps);
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if constexpr (NV > 1) channels(a.post_weight, j, post);
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[j][i] = b[j][i] * scale * (a.offset + post[i]);
                }
            }
            if (a.gate_form == MOE_GATE_TOKEN) {
                const float v = a.gate_sigmoid ? sigmoid(row_gate) : row_gate;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[j][i] *= v;
            } else if (a.gate_form == MOE_GATE_CHANNEL) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if constexpr (NV > 1) {
                        channels(a.gate, j, gate);
                        if (a.gate_sigmoid) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) gate[i] = sigmoid(gate[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[j][i] *= gate[i];
                }
            } else if (a.gate_form == MOE_GATE_ELEMENT) {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if constexpr (NV > 1) unpack8<TB>(load8_any<TB>(a.gate, n * a.gate_stride + col[j], valid[j]), g);
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[j][i] *= a.gate_sigmoid ? sigmoid(g[i]) : g[i];
                }
            }
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) r[j][i] = fmaf(a.residual_scale, r[j][i], a.block_scale * b[j][i]);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) r[j][i] = a.residual_scale * r[j][i];
        }
        if (a.residual_out) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                store8_any<TR>(a.residual_out, static_cast<size_t>(n) * a.residual_out_stride + col[j], valid[j], r[j]);
        }
        if (!a.pre_weight) continue;
        // The norm takes the sum as it is, not as a 16-bit residual_out rounds it.
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= valid[j]) r[j][i] = 0.0f;   // 0 there, but NaN with an infinite factor
                s = fmaf(r[j][i], r[j][i], s);
            }
        s = group_sum(s, slots, which);
        const float scale = 1.0f / sqrtf(s / static_cast<float>(H) + a.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (NV > 1) channels(a.pre_weight, j, pre);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] = i < valid[j] ? r[j][i] * scale * (a.offset + pre[i]) : 0.0f;
            if (a.out) store8_any<TB>(a.out, static_cast<size_t>(n) * a.out_stride + col[j], valid[j], r[j]);
            if (a.codes)
                store_e4m3(a.codes, static_cast<size_t>(n) * H + col[j], a.scales + static_cast<size_t>(n) * nb + col[j] / kFp8Block,
                           tid & 15, r[j], valid[j], flags);
            if (a.q8) store_q8(a.q8, static_cast<size_t>(n) * (H / 32) + col[j] / 32, tid & 3, r[j], valid[j] > 0, flags);
        }
    }
    if (flags) atomicOr(a.error, flags);
}

template<int TB, int TR>
hipError_t launch_norm(const NormArgs &a, hipStream_t s) {
    const int nv = a.hidden > 8192 ? 2 : 1, waves = (a.hidden + 512 * nv - 1) / (512 * nv);
    const dim3 grid(std::min(a.tokens, 256 * std::max(1, kNormWaves / waves))), block(64 * waves);
    if (nv == 1) k_block_norm<TB, TR, 1><<<grid, block, 0, s>>>(a);
    else k_block_norm<TB, TR, 2><<<grid, block, 0, s>>>(a);
    return hipGetLastError();
}

bool aligned(const void *p, size_t n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace moe

extern "C" int moe_block_norm(const moe_block_norm_args *p, void *stream) {
    constexpr int kInvalid = hipErrorInvalidValue;
    if (!p) return kInvalid;
    const moe_block_norm_args &n = *p;
    const auto is_type = [](int t) { return t == MOE_F32 || t == MOE_BF16 || t == MOE_F16; };
    if (n.hidden < 1 || n.hidden > 16384 || n.tokens < 1 || n.tokens > 65536 || !is_type(n.type) ||
        (n.residual_type != n.type && n.residual_type != MOE_F32) || !(n.eps > 0.0f) || n.eps > 3.4e38f)
        return kInvalid;
    const int es = moe::elem_bytes(n.type), rs = moe::elem_bytes(n.residual_type);
    const auto rows = [&](const void *q, int64_t stride, int size) {
        return moe::aligned(q, size) && stride >= n.hidden && stride <= (int64_t{1} << 40);
    };
    if (!rows(n.residual, n.residual_stride, rs)) return kInvalid;
    if (n.residual_out && !rows(n.residual_out, n.residual_out_stride, rs)) return kInvalid;
    if (n.block) {
        if (!rows(n.block, n.block_stride, es)) return kInvalid;
        if (n.gate_form < MOE_GATE_NONE || n.gate_form > MOE_GATE_ELEMENT) return kInvalid;
        if (n.gate_form == MOE_GATE_ELEMENT && !rows(n.gate, n.gate_stride, es)) return kInvalid;
        if ((n.gate_form == MOE_GATE_TOKEN || n.gate_form == MOE_GATE_CHANNEL) && !moe::aligned(n.gate, 4)) return kInvalid;
        if (n.post_weight && !moe::aligned(n.post_weight, 4)) return kInvalid;
    } else if (n.gate_form != MOE_GATE_NONE || n.post_weight) {
        return kInvalid;
    }
    const bool next = n.out || n.q8 || n.codes || n.scales;
    if (n.pre_weight ? !next : next) return kInvalid;
    if (!n.pre_weight && !n.residual_out) return kInvalid;   // nothing to write
    if (n.pre_weight) {
        if (!moe::aligned(n.pre_weight, 4)) return kInvalid;
        if (n.out && !rows(n.out, n.out_stride, es)) return kInvalid;
        if ((n.codes != nullptr) != (n.scales != nullptr) || (n.scales && !moe::aligned(n.scales, 4))) return kInvalid;
        if (n.q8 && (n.hidden % 32 || !moe::aligned(n.q8, 4))) return kInvalid;
        if ((n.q8 || n.codes) && !moe::aligned(n.error, 4)) return kInvalid;
    }
    moe::NormArgs a{};
    a.residual = n.residual;
    a.block = n.block;
    a.gate = n.gate;
    a.residual_out = n.residual_out;
    a.out = n.out;
    a.residual_stride = n.residual_stride;
    a.block_stride = n.block_stride;
    a.gate_stride = n.gate_stride;
    a.residual_out_stride = n.residual_out_stride;
    a.out_stride = n.out_stride;
    a.post_weight = n.post_weight;
    a.pre_weight = n.pre_weight;
    a.q8 = static_cast<uint32_t *>(n.q8);
    a.codes = static_cast<uint8_t *>(n.codes);
    a.scales = n.scales;
    a.error = n.error;
    a.eps = n.eps;
    a.offset = n.weight_offset;
    a.residual_scale = n.residual_scale;
    a.block_scale = n.block_scale;
    a.hidden = n.hidden;
    a.tokens = n.tokens;
    a.gate_form = n.block ? n.gate_form : MOE_GATE_NONE;
    a.gate_sigmoid = n.gate_sigmoid;
    const auto s = static_cast<hipStream_t>(stream);
    if (n.type == MOE_F32) return moe::launch_norm<moe::kF32, moe::kF32>(a, s);
    if (n.type == MOE_BF16)
        return n.residual_type == MOE_F32 ? moe::launch_norm<moe::kBF16, moe::kF32>(a, s) : moe::launch_norm<moe::kBF16, moe::kBF16>(a, s);
    return n.residual_type == MOE_F32 ? moe::launch_norm<moe::kF16, moe::kF32>(a, s) : moe::launch_norm<moe::kF16, moe::kF16>(a, s);
}
