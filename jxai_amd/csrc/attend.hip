// Attention of query rows over the paged 8-bit cache.
//
// A wave takes 32 rows of one sequence and kv head (row = token of the call, head within the group) against a block of 32
// tokens at a time, everything in registers:
//   S^T = K Q^T   32x32x32 int8 MFMAs: the codes of K as they lie in memory (one 16-byte load per lane and 32 dimensions)
//                 against q as two (fp32: three) signed digits of 7 bits, exact in int32
//                 (many rows: fp16 MFMAs on K converted once for the workgroup)
//   x = S * (scale of the row * scale of K's block * softmax scale), in units of log2; one scale per tile and lane
//   p = exp2(x - m), m a reference maximum of the row, at most 2^6 behind the true one
//   O^T += V^T P^T   32x32x16 fp16 MFMAs.  V's codes lie so that a lane's 16 bytes are the 16 tokens whose weights the same
//                 lane holds in the result layout of S^T: no exchange between lanes.  V's block scale goes into the
//                 weights, relative to the largest block scale seen (R), so that they stay in fp16's range.
// Each lane's column is its row, so maximum, sum and rescaling are per lane.
#include <algorithm>

#include "jxmoe_device.h"
#include "jxmoe_kv.h"

namespace jx {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int OFF = 9;        // weights are held times 2^OFF: fp16's full precision down to 2^-23 of the reference
constexpr float LOWEST = -3e38f;  // the reference of a row that has seen nothing: finite, so that differences are numbers
constexpr float LAG = 6.0f;   // the reference maximum follows when it is 2^LAG behind: 2^(OFF + LAG) < 65504

__device__ __forceinline__ float load1(const void* p, int type, int64_t i) {
    if (type == JX_TYPE_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
    return type == JX_TYPE_F16 ? f16_to_f32(v) : __uint_as_float((uint32_t)v << 16);
}

__device__ __forceinline__ uint32_t bf16_bits(float f) {  // nearest even; NaN stays NaN
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f);
}
__device__ __forceinline__ uint32_t half_bits(float f) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f); }

__device__ __forceinline__ void store1(void* p, int type, int64_t i, float v) {
    if (type == JX_TYPE_F32)
        reinterpret_cast<float*>(p)[i] = v;
    else
        reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(type == JX_TYPE_F16 ? half_bits(v) : bf16_bits(v));
}

// Four consecutive values; vec: their place is aligned to four values
__device__ __forceinline__ void store4(void* p, int type, int64_t i, bool vec, float4 v) {
    if (vec && type == JX_TYPE_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = v;
    } else if (vec) {
        uint2 u;
        if (type == JX_TYPE_F16)
            u = make_uint2(half_bits(v.x) | half_bits(v.y) << 16, half_bits(v.z) | half_bits(v.w) << 16);
        else
            u = make_uint2(bf16_bits(v.x) | bf16_bits(v.y) << 16, bf16_bits(v.z) | bf16_bits(v.w) << 16);
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = u;
    } else {
        store1(p, type, i, v.x), store1(p, type, i + 1, v.y), store1(p, type, i + 2, v.z), store1(p, type, i + 3, v.w);
    }
}

// 16 consecutive values of a row
__device__ __forceinline__ void load16(const void* p, int type, int64_t i, bool vec, float (&v)[16]) {
    if (vec && type == JX_TYPE_F32) {
        const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 f = s[k];
            v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
        }
    } else if (vec) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint4 u = s[k];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                v[8 * k + 2 * m] = type == JX_TYPE_F16 ? f16_to_f32(w[m] & 0xFFFFu) : __uint_as_float(w[m] << 16);
                v[8 * k + 2 * m + 1] = type == JX_TYPE_F16 ? f16_to_f32(w[m] >> 16) : __uint_as_float(w[m] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = load1(p, type, i + k);
    }
}

// tanh, relative error under 1e-6 near zero and absolute under 1e-7 elsewhere
__device__ __forceinline__ float tanh_fast(float z) {
    const float a = __builtin_fabsf(z), z2 = z * z;
    const float e = __builtin_amdgcn_exp2f(-2.0f * LOG2E * a);
    const float big = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    // the series of tanh to z^9
    float s = __builtin_fmaf(z2, 62.0f / 2835.0f, -17.0f / 315.0f);
    s = __builtin_fmaf(z2, s, 2.0f / 15.0f);
    s = __builtin_fmaf(z2, s, -1.0f / 3.0f);
    const float small = __builtin_fmaf(a * z2, s, a);
    return __builtin_copysignf(a < 0.25f ? small : big, z);
}

__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ float lane_of(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

// (v of the lane 32 below or its own, v of the lane 32 above or its own): one of the two is the other half's.  16: of each 32 lanes
__device__ __forceinline__ float2 both32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 both16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Over the lanes of a row: lane + 32 (and + 16, where 16 lanes hold the rows)
template <int NR>
__device__ __forceinline__ float row_max(float v) {
    const float2 a = both32(v);
    v = fmaxf(a.x, a.y);
    if constexpr (NR == 16) {
        const float2 b = both16(v);
        v = fmaxf(b.x, b.y);
    }
    return v;
}
template <int NR>
__device__ __forceinline__ float row_sum(float v) {
    const float2 a = both32(v);
    v = a.x + a.y;
    if constexpr (NR == 16) {
        const float2 b = both16(v);
        v = b.x + b.y;
    }
    return v;
}

typedef float v4f __attribute__((ext_vector_type(4)));

// What differs between a wave that takes 32 rows and one that takes up to 16 (half the registers and arithmetic for the same
// codes, so twice the waves: the form for single tokens).  col: the lane's row; g: its part of the others' dimension.
//   result of K Q^T: register x holds token token(x) + 4 g; of V^T P^T: register x of tile i holds dimension DI * i + dim(x) + 4 g
template <int NR, int DT>
struct Form;
template <int DT>
struct Form<32, DT> {
    typedef v16i Acc;
    typedef v16f Out;
    static constexpr int STEPS = DT, X = 16, TILES = DT, DI = 32, ACCS = 1;  // ACCS: result tiles of 32 tokens
    static __device__ constexpr int token(int x) { return 8 * (x >> 2) + (x & 3); }
    static __device__ constexpr int dim(int x) { return 8 * (x >> 2) + (x & 3); }
    static __device__ __forceinline__ int chunk(int j, int g) { return 2 * j + g; }  // of 16 dimensions
    static __device__ __forceinline__ int k_at(int j, int g, int col) { return (2 * j + g) * 512 + col * 16; }
    static __device__ __forceinline__ int v_at(int j, int g, int col) { return (g * 32 * DT + 32 * j + col) * 16; }
    static __device__ __forceinline__ Acc scores(v4i k, v4i q, Acc c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(k, q, c, 0, 0, 0); }
};
template <int DT>
struct Form<16, DT> {
    typedef v4i Acc;
    typedef v4f Out;
    static constexpr int STEPS = (DT + 1) / 2, X = 8, TILES = 2 * DT, DI = 16, ACCS = 2;
    static __device__ constexpr int token(int x) { return 16 * (x >> 2) + (x & 3); }
    static __device__ constexpr int dim(int x) { return x; }
    static __device__ __forceinline__ int chunk(int j, int g) { return 4 * j + g; }
    // (the last step of an odd DT has two chunks: the other lanes read the same ones, against zeros of q)
    static __device__ __forceinline__ int k_chunk(int j, int g) { return DT % 2 && j == STEPS - 1 ? 4 * j + (g & 1) : 4 * j + g; }
    static __device__ __forceinline__ Acc scores(v4i k, v4i q, Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q, c, 0, 0, 0); }
};

template <int NR, int DT>
using AccOf = typename Form<NR, DT>::Acc;
template <int NR, int DT, int ND>
using Scores = AccOf<NR, DT>[ND][Form<NR, DT>::ACCS];
template <int NR, int DT, int ND>
using Digits = v4i[ND][Form<NR, DT>::STEPS];
template <int NR, int DT>
using Keys = v4i[Form<NR, DT>::ACCS][Form<NR, DT>::STEPS];

// The lane's values of q: the 16 dimensions of chunk(j, g) of its row
template <int NR, int DT>
using Raw = float[Form<NR, DT>::STEPS][16];
template <int NR, int DT>
__device__ __forceinline__ void load_q(const AttendArgs& a, int row, int head, int g, bool valid, Raw<NR, DT>& v) {
    typedef Form<NR, DT> F;
    const int64_t at = (int64_t)row * a.q_stride + (int64_t)head * a.c.D;
#pragma unroll
    for (int j = 0; j < F::STEPS; ++j) {
        if (valid && F::chunk(j, g) < 2 * DT) {
            load16(a.q, a.type, at + 16 * F::chunk(j, g), a.q_vec, v[j]);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[j][k] = 0.0f;
        }
    }
}

// Byte 0 of four words
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
    return lo | hi;
}

// ND signed digits of it in MFMA operand order, 127 times the top digit's unit for the row's largest value.  qs: the value of one
// unit of the last digit, NaN where the row has a value that is not finite.
//   u = rint(v * TOP / amax) + 64 (1 + 128): added to 1.5 2^23 by the multiply-add that forms it, u is in the low mantissa bits;
//   its groups of 7 bits are the lower digits + 64, what is above them the top digit.
template <int NR, int DT, int ND>
__device__ __forceinline__ void digits(const Raw<NR, DT>& v, bool flip, Digits<NR, DT, ND>& qd, float& qs) {
    typedef Form<NR, DT> F;
    constexpr float TOP = ND == 2 ? 127.0f * 128.0f : 127.0f * 16384.0f;
    constexpr float MAGIC = 12582912.0f + (ND == 2 ? 64.0f : 64.0f + 64.0f * 128.0f);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(v[j][k]) & 0x7FFFFFFFu);  // orders NaN and infinity last
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    if constexpr (NR == 16) top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    const bool finite = top < 0x7F800000u;
    // rows below 2^-100 count as zero: TOP / amax stays finite
    const bool zero = top < 0x0D800000u;
    const float amax = __uint_as_float(top);
    const float inv = finite && !zero ? (flip ? -TOP : TOP) / amax : 0.0f;
    qs = !finite ? __uint_as_float(0x7FC00000u) : zero ? 0.0f : amax / TOP;
#pragma unroll
    for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(__builtin_fmaf(v[j][k + i], inv, MAGIC));
#pragma unroll
            for (int n = ND - 1; n > 0; --n) {
                // a byte d + 64 (0 .. 127) -> d: bit 6 flipped, and the sign where it is then set
                const uint32_t y = (pack4(u[0], u[1], u[2], u[3]) & 0x7F7F7F7Fu) ^ 0x40404040u;
                qd[n][j][k >> 2] = (int)(y | (y & 0x40404040u) << 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] >>= 7;
            }
            qd[0][j][k >> 2] = (int)pack4(u[0], u[1], u[2], u[3]);
        }
}

// The same as one (fp32: two) fp16 values each, with the row's largest between 2^4 and 2^5: the form for K in fp16 (k_attend_rows).
// F16 and BF16 are held whole, except below 2^-18 of the row's largest; fp32 in 22 bits.  piece u of step j: dimensions 8 u .. + 7
template <int DT, int ND>
__device__ __forceinline__ void halves(const Raw<32, DT>& v, bool flip, h8 (&qh)[ND - 1][DT][2], float& qs) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(v[j][k]) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    const bool finite = top < 0x7F800000u, zero = top < 0x0D800000u;
    const int e = (int)(top >> 23) - 127 - 4;  // the row in units of 2^e
    const float inv = finite && !zero ? __uint_as_float((uint32_t)(127 - e) << 23) : 0.0f;
    qs = !finite ? __uint_as_float(0x7FC00000u) : zero ? 0.0f : __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float u = v[j][k] * (flip ? -inv : inv);
            qh[0][j][k >> 3][k & 7] = (_Float16)u;
            if constexpr (ND == 3) qh[1][j][k >> 3][k & 7] = (_Float16)(u - (float)(_Float16)u);
        }
}

// What a wave carries for its rows.
template <int NR, int DT>
struct Carry {
    typename Form<NR, DT>::Out o[Form<NR, DT>::TILES];
    float m, l;  // of the lane's row: reference maximum (log2), sum of the weights of the lane's tokens
    float R;     // largest scale of V's blocks so far
};

template <int NR, int DT>
__device__ __forceinline__ void carry_init(Carry<NR, DT>& s) {
#pragma unroll
    for (auto& o : s.o) o = typename Form<NR, DT>::Out{};
    s.m = LOWEST;
    s.l = 0.0f;
    s.R = 0.0f;
}

template <int NR, int DT>
__device__ __forceinline__ void carry_scale(Carry<NR, DT>& s, float f) {
#pragma unroll
    for (auto& o : s.o)
#pragma unroll
        for (int k = 0; k < (NR == 32 ? 16 : 4); ++k) o[k] *= f;
}

__device__ __forceinline__ h8 codes_to_half(uint32_t w0, uint32_t w1) {
    const h2v one = {(_Float16)1.0f, (_Float16)1.0f}, bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return cvt8(w0, w1, 0xFFFFFFFFu, 0x80808080u, one, bias);  // 1024 + (code + 128) - 1152
}

// S^T of one block of 32 tokens, digit by digit.  kc: [result tile][step]
template <int NR, int DT, int ND>
__device__ __forceinline__ void scores(Scores<NR, DT, ND>& acc, const Digits<NR, DT, ND>& qd,
                                       const Keys<NR, DT>& kc) {
    typedef Form<NR, DT> F;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int t = 0; t < F::ACCS; ++t) acc[n][t] = typename F::Acc{};
#pragma unroll
    for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
        for (int t = 0; t < F::ACCS; ++t)
#pragma unroll
            for (int n = 0; n < ND; ++n) acc[n][t] = F::scores(kc[t][j], qd[n][j], acc[n][t]);
}

// The weights of a lane's row and tokens as operand of the product with V, in the order of V's bytes; e: what their rounding
// left (fp32: 22 bits in all).
template <int NR, int ND>
struct Weights {
    h8 p[NR / 16], e[ND == 3 ? NR / 16 : 1];
};

// S^T as floats in units of the last digit
template <int NR, int DT, int ND>
__device__ __forceinline__ void score_values(const Scores<NR, DT, ND>& acc, float (&x)[Form<NR, DT>::X]) {
    typedef Form<NR, DT> F;
    constexpr int X = F::X, PER = X / F::ACCS;
#pragma unroll
    for (int i = 0; i < X; ++i) {
        const int t = i / PER, k = i % PER;
        // |acc| <= 127 * 127 * 256: two digits fit an int32
        if constexpr (ND == 2)
            x[i] = (float)(int)(((uint32_t)acc[0][t][k] << 7) + (uint32_t)acc[1][t][k]);
        else
            x[i] = __builtin_fmaf((float)acc[0][t][k], 16384.0f, (float)(int)(((uint32_t)acc[1][t][k] << 7) + (uint32_t)acc[2][t][k]));
    }
}

// The scores x (in units of qs * ks) of a block whose tokens begin at t0, capped, biased and masked: x * c is the exponent of 2
// afterwards.  Returns the row's largest.  lo / hi: the lane's row sees tokens lo .. hi - 1 (masked: whether to look).
template <int NR, int DT, bool EXT>
__device__ __forceinline__ float see_scores(const AttendArgs& a, float (&x)[Form<NR, DT>::X], float& c, float qs, float slope, int pos, float ks,
                                            int t0, int g, int lo, int hi, bool masked) {
    typedef Form<NR, DT> F;
    constexpr int X = F::X;
    // (c is kept above 0, so that a masked -inf stays what it is; the sign of the softmax scale is in q)
    c = qs * ks * (EXT ? a.scale : a.scale2);
    c = c < 1e-30f ? 1e-30f : c;
    if constexpr (EXT) {
        const float inv = a.cap > 0.0f ? 1.0f / a.cap : 0.0f, d0 = (float)(t0 + 4 * g - pos);
#pragma unroll
        for (int i = 0; i < X; ++i) {
            x[i] *= c;
            if (a.cap > 0.0f) x[i] = a.cap * tanh_fast(x[i] * inv);
            x[i] = __builtin_fmaf(slope, d0 + (float)F::token(i), x[i]);
        }
        c = LOG2E;
    }
    if (masked) {
        const int l0 = lo - t0 - 4 * g, h0 = hi - t0 - 4 * g;
#pragma unroll
        for (int i = 0; i < X; ++i) x[i] = F::token(i) >= l0 && F::token(i) < h0 ? x[i] : -__builtin_inff();
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < X; ++i) top = fmaxf(top, x[i]);
    return top * c;
}

// The reference maximum after scores up to `top` (of the lane's tokens)
template <int NR, int DT>
__device__ __forceinline__ void follow(Carry<NR, DT>& s, float top) {
    top = row_max<NR>(top);
    if (__any(top > s.m + LAG)) {
        const float m = fmaxf(s.m, top), f = __builtin_amdgcn_exp2f(s.m - m);
        s.m = m;
        s.l *= f;
        carry_scale(s, f);
    }
}
// R after a block of scale vs.  One of NaN makes every row NaN that sees a token of the block (x: its scores).
template <int NR, int DT>
__device__ __forceinline__ void follow_value(Carry<NR, DT>& s, const float (&x)[Form<NR, DT>::X], float& vs) {
    if (!(vs <= s.R)) {
        if (vs > s.R) {
            carry_scale(s, s.R * __builtin_amdgcn_rcpf(vs));
            s.R = vs;
        } else {
            bool sees = false;
#pragma unroll
            for (float v : x) sees |= v != -__builtin_inff();
            s.l += sees ? vs : 0.0f;
            vs = 0.0f;
        }
    }
}

// The weights of a block.  V's scale relative to R goes into the exponent and out of the sum again.  (A block of zeros, whose
// scale is 0, may weigh anything; 2^-100 of R is far below what the weights' fp16 holds.)
template <int NR, int DT, int ND>
__device__ __forceinline__ Weights<NR, ND> weights(Carry<NR, DT>& s, float (&x)[Form<NR, DT>::X], float c, float vs) {
    constexpr int X = Form<NR, DT>::X;
    const float vr = vs == 0.0f ? 1.0f : fmaxf(vs * __builtin_amdgcn_rcpf(s.R), 0x1p-100f);
    const float ref = s.m - ((float)OFF + __builtin_amdgcn_logf(vr));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < X; ++i) {
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -ref));
        sum += x[i];
    }
    s.l = __builtin_fmaf(sum, __builtin_amdgcn_rcpf(vr), s.l);
    // 32 rows: token 8 a + 4 g + b is register 4 a + b here and byte 8 (a & 1) + 4 (a >> 1) + b of V.  16 rows: in order
    Weights<NR, ND> w;
#pragma unroll
    for (int i = 0; i < X; ++i) {
        const int o = NR == 32 ? (i >> 2) & 1 : 0, at = NR == 32 ? 4 * (i >> 3) + (i & 3) : i;
        w.p[o][at] = (_Float16)x[i];
        if constexpr (ND == 3) w.e[o][at] = (_Float16)(x[i] - (float)w.p[o][at]);
    }
    return w;
}

template <int NR>
__device__ __forceinline__ auto value_mfma(h8 v, h8 p, typename Form<NR, 1>::Out o) {
    if constexpr (NR == 32)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p, o, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o, 0, 0, 0);
}

// Their product with V from its codes in registers
template <int NR, int DT, int ND>
__device__ __forceinline__ void add_values(Carry<NR, DT>& s, const Weights<NR, ND>& w, const v4i (&vc)[DT]) {
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        if constexpr (NR == 32) {
            const h8 v0 = codes_to_half((uint32_t)vc[i][0], (uint32_t)vc[i][1]);
            const h8 v1 = codes_to_half((uint32_t)vc[i][2], (uint32_t)vc[i][3]);
            s.o[i] = value_mfma<NR>(v0, w.p[0], s.o[i]);
            s.o[i] = value_mfma<NR>(v1, w.p[1], s.o[i]);
            if constexpr (ND == 3) {
                s.o[i] = value_mfma<NR>(v0, w.e[0], s.o[i]);
                s.o[i] = value_mfma<NR>(v1, w.e[1], s.o[i]);
            }
        } else {
            // registers 0 .. 3 are tokens 4 g + b, 4 .. 7 tokens 16 + 4 g + b: of a piece (h, d) of V the eight bytes from
            // 8 (g >> 1) on, h = g & 1.  The lane loaded all 16 bytes of piece h of dimension 32 i + 16 (g >> 1) + col: the
            // halves of the wave exchange what belongs to the other's 16 dimensions.
            const auto r0 = __builtin_amdgcn_permlane32_swap((uint32_t)vc[i][0], (uint32_t)vc[i][2], false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap((uint32_t)vc[i][1], (uint32_t)vc[i][3], false, false);
            const h8 v0 = codes_to_half(r0[0], r1[0]), v1 = codes_to_half(r0[1], r1[1]);
            s.o[2 * i] = value_mfma<NR>(v0, w.p[0], s.o[2 * i]);
            s.o[2 * i + 1] = value_mfma<NR>(v1, w.p[0], s.o[2 * i + 1]);
            if constexpr (ND == 3) {
                s.o[2 * i] = value_mfma<NR>(v0, w.e[0], s.o[2 * i]);
                s.o[2 * i + 1] = value_mfma<NR>(v1, w.e[0], s.o[2 * i + 1]);
            }
        }
    }
}

// The blocks of up to 64 tiles, one per lane
struct Blocks {
    int k, v;       // block numbers
    float ks, vs;   // scales
};
__device__ __forceinline__ int page_of(const AttendArgs& a, int slot, int tile, bool valid) {
    return valid ? a.c.table[(int64_t)slot * a.c.max_pages + (tile >> a.c.blocks_shift)] : 0;
}
__device__ __forceinline__ Blocks blocks_of(const AttendArgs& a, int kvh, int page, int tile, bool valid) {
    Blocks b = {0, 0, 0.0f, 0.0f};
    if (valid) {
        const bool bad = page < 0 || page >= a.c.n_pages;
        page = bad ? 0 : page;
        const int blk = tile & ((1 << a.c.blocks_shift) - 1);
        b.k = a.c.block_index(page, 0, kvh, blk);
        b.v = a.c.block_index(page, 1, kvh, blk);
        b.ks = a.c.scales[b.k];
        b.vs = a.c.scales[b.v];
        if (bad) {
            b.ks = b.vs = __uint_as_float(0x7FC00000u);
            atomicOr(a.c.status, JX_KV_BAD_PAGE);
        }
    }
    return b;
}

// A wave's rows against `count` tiles, first + i * step.  Everything that waits for memory is asked for as early as its address is
// known: pages, then q, then scales and the first block, and q's digits are formed while that arrives.  In the loop a
// block's registers are loaded again as soon as its products are issued: the next K arrives behind the weights and the
// product with V, the next V behind the next scores.  (Two full sets of registers spilled at 128 dimensions.)
template <int NR, int DT, int ND, bool EXT, bool ONCE>
__device__ __forceinline__ void attend_tiles(Carry<NR, DT>& cy, const AttendArgs& a, const KvSeq& s, int kvh, int row, int head, bool valid,
                                             int pos, int first, int step, int count, int whole_lo, int whole_hi) {
    typedef Form<NR, DT> F;
    const int lane = threadIdx.x & 63, g = lane / NR, col = lane % NR;
    const int hi = a.causal ? min(s.len, pos + 1) : s.len, lo = a.window ? max(0, pos - a.window + 1) : 0;
    const int64_t bytes = (int64_t)KV_BLOCK * 32 * DT;
    auto ld = [](const int8_t* p) {  // (blocks that one wave alone reads: without a place in the caches)
        const v4i* q = reinterpret_cast<const v4i*>(p);
        return ONCE ? __builtin_nontemporal_load(q) : *q;
    };
    Blocks bl;
    Keys<NR, DT> k;
    v4i v[DT];
    auto fetch_k = [&](int i) {
        const int8_t* p = a.c.codes + lane_of(bl.k, i) * bytes;
#pragma unroll
        for (int j = 0; j < F::STEPS; ++j)
#pragma unroll
            for (int t = 0; t < F::ACCS; ++t) {
                if constexpr (NR == 32)
                    k[t][j] = ld(p + F::k_at(j, g, col));
                else
                    k[t][j] = ld(p + F::k_chunk(j, g) * 512 + (16 * t + col) * 16);
            }
    };
    auto fetch_v = [&](int i) {
        const int8_t* p = a.c.codes + lane_of(bl.v, i) * bytes;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            if constexpr (NR == 32)
                v[j] = ld(p + F::v_at(j, g, col));
            else
                v[j] = ld(p + ((g & 1) * 32 * DT + 32 * j + 16 * (g >> 1) + col) * 16);
        }
    };
    int page = page_of(a, s.slot, first + lane * step, lane < count);
    Raw<NR, DT> raw;
    load_q<NR, DT>(a, row, head, g, valid, raw);
    const float slope = EXT && a.alibi ? a.alibi[head] : 0.0f;
    bl = blocks_of(a, kvh, page, first + lane * step, lane < count);
    if (count > 0) {
        fetch_k(0);
        fetch_v(0);
    }
    Digits<NR, DT, ND> qd;
    float qs;
    digits<NR, DT, ND>(raw, a.flip, qd, qs);
    for (int b0 = 0; b0 < count; b0 += 64) {
        const int n = min(64, count - b0);
        if (b0) {
            const int mine = first + (b0 + lane) * step;
            bl = blocks_of(a, kvh, page_of(a, s.slot, mine, lane < n), mine, lane < n);
            fetch_k(0);
            fetch_v(0);
        }
        for (int i = 0; i < n; ++i) {
            Scores<NR, DT, ND> acc;
            scores<NR, DT, ND>(acc, qd, k);
            if (i + 1 < n) fetch_k(i + 1);
            const int t0 = (first + (b0 + i) * step) * KV_BLOCK;
            float x[F::X];
            score_values<NR, DT, ND>(acc, x);
            float c, vs = lane_of(bl.vs, i);
            follow(cy, see_scores<NR, DT, EXT>(a, x, c, qs, slope, pos, lane_of(bl.ks, i), t0, g, lo, hi,
                                               t0 < whole_lo || t0 + KV_BLOCK > whole_hi));
            follow_value(cy, x, vs);
            const auto w = weights<NR, DT, ND>(cy, x, c, vs);
            add_values<NR, DT, ND>(cy, w, v);
            if (i + 1 < n) fetch_v(i + 1);
        }
    }
}

// The sums of the lane's row as floats at o (16-byte aligned), times f
template <int NR, int DT>
__device__ __forceinline__ void put_sums(const Carry<NR, DT>& cy, float* o, int g, float f) {
    typedef Form<NR, DT> F;
#pragma unroll
    for (int i = 0; i < F::TILES; ++i)
#pragma unroll
        for (int k = 0; k < (NR == 32 ? 16 : 4); k += 4)
            *reinterpret_cast<float4*>(o + F::DI * i + F::dim(k) + 4 * g) =
                make_float4(cy.o[i][k] * f, cy.o[i][k + 1] * f, cy.o[i][k + 2] * f, cy.o[i][k + 3] * f);
}
// The same as the call's type at element `at` of out
template <int NR, int DT>
__device__ __forceinline__ void put_out(const Carry<NR, DT>& cy, const AttendArgs& a, int64_t at, int g, float f) {
    typedef Form<NR, DT> F;
#pragma unroll
    for (int i = 0; i < F::TILES; ++i)
#pragma unroll
        for (int k = 0; k < (NR == 32 ? 16 : 4); k += 4) {
            const float4 y = make_float4(cy.o[i][k] * f, cy.o[i][k + 1] * f, cy.o[i][k + 2] * f, cy.o[i][k + 3] * f);
            store4(a.out, a.type, at + F::DI * i + F::dim(k) + 4 * g, a.out_vec, y);
        }
}

// The tiles of 32 tokens that a row tile of a sequence sees, and how they are divided.
struct Range {
    int begin, tiles;  // first tile, count
    int per, n;        // tiles per split, splits
    int base;          // position of the call's first row
};
__device__ __forceinline__ Range range_of(const AttendArgs& a, const KvSeq& s, int r0, int nr) {
    Range g;
    g.base = s.len - s.n;
    const int i0 = r0 / a.G, i1 = (r0 + nr - 1) / a.G;
    const int hi = a.causal ? min(s.len, g.base + i1 + 1) : s.len;
    const int lo = a.window ? max(0, g.base + i0 - a.window + 1) : 0;
    g.begin = lo / KV_BLOCK;
    g.tiles = hi > lo ? (hi + KV_BLOCK - 1) / KV_BLOCK - g.begin : 0;
    g.n = max(1, min(a.splits, (g.tiles + a.chunk - 1) / a.chunk));
    g.per = max(1, (g.tiles + g.n - 1) / g.n);
    g.n = max(1, (g.tiles + g.per - 1) / g.per);
    return g;
}

// Waves of a workgroup: wide heads need more than 256 registers, and LDS for the join.
__host__ __device__ constexpr int waves_of(int dt) { return dt <= 4 ? 8 : 4; }

// Up to 32 rows over a short sequence: a workgroup for each sequence and kv head (blockIdx.x = sequence * H + kv head), whose waves
// take its tiles in turn and join in LDS.  One launch: the form for latency.
template <int NR, int DT, int ND, bool EXT>
__global__ __launch_bounds__(64 * waves_of(DT)) void k_attend(const AttendArgs a) {
    extern __shared__ float lds[];
    constexpr int W = waves_of(DT);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, gl = lane / NR, col = lane % NR, D = a.c.D;
    const int kvh = blockIdx.x % a.c.H, seq = blockIdx.x / a.c.H;
    const int failed = *a.c.status;
    const KvSeq s = kv_seq(a.c, a.b, seq);
    const int rows = s.n * a.G;
    if (rows == 0) return;
    const Range g = range_of(a, s, 0, rows);
    const int r = min(col, rows - 1), head = kvh * a.G + r % a.G, row = s.row0 + r / a.G, pos = g.base + r / a.G;
    // tiles that every row sees whole need no mask: hi of the first row, lo of the last
    const int whole_hi = a.causal ? min(s.len, g.base + 1) : s.len, whole_lo = a.window ? max(0, g.base + s.n - a.window) : 0;
    Carry<NR, DT> cy;
    carry_init(cy);
    attend_tiles<NR, DT, ND, EXT, false>(cy, a, s, kvh, row, head, col < rows, pos, g.begin + wave, W, (g.tiles - wave + W - 1) / W,
                                         whole_lo, whole_hi);

    // the waves' sums: [W][rows_cap][D], then [W][rows_cap] of the maximum and the sum of weights
    float* so = lds;
    float2* sm = reinterpret_cast<float2*>(lds + (size_t)W * a.rows_cap * D);
    cy.l = row_sum<NR>(cy.l);
    if (col < rows) {
        put_sums(cy, so + ((size_t)wave * a.rows_cap + col) * D, gl, cy.R);
        if (gl == 0) sm[wave * a.rows_cap + col] = make_float2(cy.m, cy.l);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * D; i += 64 * W) {
        const int rr = i / D, d = i - rr * D;
        float m = -__builtin_inff(), o = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, sm[w * a.rows_cap + rr].x);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 ml = sm[w * a.rows_cap + rr];
            const float f = ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
            l = __builtin_fmaf(f, ml.y, l);
            o = __builtin_fmaf(f, so[((size_t)w * a.rows_cap + rr) * D + d], o);
        }
        float y = l == 0.0f ? 0.0f : o / l;
        if (failed) y = __uint_as_float(0x7FC00000u);
        store1(a.out, a.type, (int64_t)(s.row0 + rr / a.G) * a.out_stride + (int64_t)(kvh * a.G + rr % a.G) * D + d, y);
    }
}

// ---------------------------------------------------------------- many rows: K and V through LDS

constexpr int ROWS_W = 4;  // waves; two workgroups share a CU (up to 128 dimensions)
constexpr int STAGE = 2;   // blocks of 32 tokens in LDS at a time

// 32 rows per wave, four waves against the same blocks.  A stage of two blocks goes through registers into one of two LDS buffers
// as fp16, K and V in the order that the products read (16 bytes per lane in a row), converted once for all waves.  While a
// stage is worked on, the next one is written to LDS and the two behind that are on their way; one barrier per stage.
// K Q^T is fp16 here, not digits: the vector unit is what bounds the loop, and joining and converting two digits' sums costs
// it 32 of about 150 instructions per block.
// blockIdx.x = ((sequence * splits + split) * row_tiles + row tile from the last) * H + kv head: the longest rows of a
// causal prompt first, and the row tiles of 8 kv heads each on an XCD of their own, whose L2 keeps the head's K and V.
template <int DT, int ND, bool EXT>
__global__ __launch_bounds__(64 * ROWS_W, DT <= 4 ? 2 : 1) void k_attend_rows(const AttendArgs a) {
    constexpr int W = ROWS_W, KB = 1024 * DT, HB = 2 * KB, BUF = STAGE * 2 * HB;  // bytes of a block, in fp16, of a buffer
    constexpr int LOADS = (2 * STAGE * DT + W - 1) / W;  // of 1 KB per wave and stage
    extern __shared__ uint4 lds4[];
    __shared__ Blocks ring[128];
    uint8_t* lds = reinterpret_cast<uint8_t*>(lds4);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, gl = lane >> 5, col = lane & 31;
    int item = blockIdx.x;
    const int kvh = item % a.c.H;
    item /= a.c.H;
    const int rt = a.row_tiles - 1 - item % a.row_tiles;
    item /= a.row_tiles;
    const int split = item % a.splits, seq = item / a.splits;
    const int failed = *a.c.status;
    const KvSeq s = kv_seq(a.c, a.b, seq);
    const int rows = s.n * a.G, r0 = rt * a.tile_rows;
    if (r0 >= rows) return;
    const int nr = min(a.tile_rows, rows - r0);
    const Range g = range_of(a, s, r0, nr);
    if (split >= g.n) return;
    // the wave's rows
    const int w0 = r0 + 32 * wave, wn = min(32, r0 + nr - w0);  // (wn <= 0: a wave without rows only moves the blocks)
    const int r = min(w0 + col, rows - 1), head = kvh * a.G + r % a.G, row = s.row0 + r / a.G, pos = g.base + r / a.G;
    const int hi = a.causal ? min(s.len, pos + 1) : s.len, lo = a.window ? max(0, pos - a.window + 1) : 0;
    const int p0 = g.base + min(w0, rows - 1) / a.G, p1 = g.base + min(w0 + 31, rows - 1) / a.G;
    // tokens that some row of the wave sees, and that every row sees
    const int some_hi = wn <= 0 ? 0 : a.causal ? min(s.len, p1 + 1) : s.len, some_lo = a.window ? max(0, p0 - a.window + 1) : 0;
    const int whole_hi = a.causal ? min(s.len, p0 + 1) : s.len, whole_lo = a.window ? max(0, p1 - a.window + 1) : 0;

    Carry<32, DT> cy;
    carry_init(cy);
    const int first = g.begin + split * g.per, count = min(g.tiles, (split + 1) * g.per) - split * g.per;
    // load u = wave + i * W of a stage: K of its blocks, then V, a kilobyte each
    typedef uint4 Load[LOADS];
    Load in0, in1;  // of even and odd stages
    auto fetch = [&](Load& in, int t, auto block_of) {  // the stage from tile t on
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int u = wave + i * W;
            if (u >= 2 * STAGE * DT) break;
            const int which = u >= STAGE * DT, v = u - which * STAGE * DT;
            const int block = block_of(min(t + v / DT, count - 1), which);
            in[i] = ld16(a.c.codes + (int64_t)block * KB + (v % DT) * 1024 + lane * 16);
        }
    };
    auto put = [&](const Load& in, int buf) {
        uint8_t* to = lds + buf * BUF;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int u = wave + i * W;
            if (u >= 2 * STAGE * DT) break;
            const int which = u >= STAGE * DT, v = u - which * STAGE * DT, b = v / DT, kb = v % DT;
            // K: the lane's 16 bytes are dimensions 16 h .. of step kb; V: piece (h, d).  Eight for each of two products
            const int piece = kb * 64 + lane, h = piece / (32 * DT), d = piece % (32 * DT);
            h8* o = reinterpret_cast<h8*>(to + (2 * b + which) * HB) + (which ? (d >> 5) * 128 + h * 32 + (d & 31) : kb * 128 + lane);
            o[0] = codes_to_half(in[i].x, in[i].y);
            o[64] = codes_to_half(in[i].z, in[i].w);
        }
    };
    // blocks and scales of 128 tiles around the current one: wave 0 looks the next 64 up, a step per stage
    auto keep = [&](int t, const Blocks& b) { ring[(t + lane) & 127] = b; };
    auto ring_block = [&](int t, int which) { return __builtin_amdgcn_readfirstlane(which ? ring[t & 127].v : ring[t & 127].k); };
    auto look = [&](int t) { return page_of(a, s.slot, first + t + lane, t + lane < count); };
    auto find = [&](int t, int page) { return blocks_of(a, kvh, page, first + t + lane, t + lane < count); };

    h8 qh[ND - 1][DT][2];
    float qs, slope = 0.0f;
    int page = look(0);
    Blocks bl;
    {
        Raw<32, DT> raw;
        load_q<32, DT>(a, row, head, gl, w0 + col < r0 + nr, raw);
        if (EXT && a.alibi) slope = a.alibi[head];
        bl = find(0, page);
        if (count > 0) fetch(in0, 0, [&](int t, int which) { return which ? lane_of(bl.v, t) : lane_of(bl.k, t); });
        halves<DT, ND>(raw, a.flip, qh, qs);
    }
    auto first_block = [&](int t, int which) { return which ? lane_of(bl.v, t) : lane_of(bl.k, t); };
    if (wave == 0) keep(0, bl);
    if (STAGE < count) fetch(in1, STAGE, first_block);
    if (count > 0) put(in0, 0);
    if (2 * STAGE < count) fetch(in0, 2 * STAGE, first_block);
    __syncthreads();
    auto scale_of = [&](int t, bool v) {
        const Blocks& b = ring[t & 127];
        return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v ? b.vs : b.ks)));
    };
    constexpr int VH = DT < 4 ? 2 * DT : 8;  // pieces of V that are read ahead of the exponentials
    auto stage = [&](int t, int buf, Load& in) {  // `in`: holds the next stage
        if (t + STAGE < count) put(in, buf ^ 1);
        if (t + 3 * STAGE < count) fetch(in, t + 3 * STAGE, ring_block);
        if (wave == 0) {  // (the steps are one stage apart: each waits for what the one before asked for)
            const int from = (t & ~63) + 64, at = t & 63;
            if (from < count) {
                if (at == 0) page = look(from);
                if (at == STAGE) bl = find(from, page);
                if (at == 2 * STAGE) keep(from, bl);
            }
        }
#pragma unroll
        for (int b = 0; b < STAGE; ++b) {
            const int t0 = (first + t + b) * KV_BLOCK;
            if (t + b >= count || t0 >= some_hi || t0 + KV_BLOCK <= some_lo) continue;
            const h8* from = reinterpret_cast<const h8*>(lds + buf * BUF + 2 * b * HB) + lane;
            const float ks = scale_of(t + b, false);
            float vs = scale_of(t + b, true), c;
            h8 k[2 * DT], v[2 * DT];
#pragma unroll
            for (int j = 0; j < 2 * DT; ++j) k[j] = from[j * 64];
            __builtin_amdgcn_sched_barrier(0);
            v16f acc = {};
#pragma unroll
            for (int j = 0; j < 2 * DT; ++j) {
                acc = value_mfma<32>(k[j], qh[0][j >> 1][j & 1], acc);
                if constexpr (ND == 3) acc = value_mfma<32>(k[j], qh[1][j >> 1][j & 1], acc);
            }
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = acc[i];
            follow(cy, see_scores<32, DT, EXT>(a, x, c, qs, slope, pos, ks, t0, gl, lo, hi, t0 < whole_lo || t0 + KV_BLOCK > whole_hi));
            follow_value(cy, x, vs);
#pragma unroll
            for (int i = 0; i < VH; ++i) v[i] = from[HB / 16 + i * 64];
            __builtin_amdgcn_sched_barrier(0);
            const auto w = weights<32, DT, ND>(cy, x, c, vs);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                if (2 * i + VH < 2 * DT)
                    v[2 * i + VH] = from[HB / 16 + (2 * i + VH) * 64], v[2 * i + VH + 1] = from[HB / 16 + (2 * i + VH + 1) * 64];
                cy.o[i] = value_mfma<32>(v[2 * i], w.p[0], cy.o[i]);
                cy.o[i] = value_mfma<32>(v[2 * i + 1], w.p[1], cy.o[i]);
                if constexpr (ND == 3) {
                    cy.o[i] = value_mfma<32>(v[2 * i], w.e[0], cy.o[i]);
                    cy.o[i] = value_mfma<32>(v[2 * i + 1], w.e[1], cy.o[i]);
                }
            }
        }
        __syncthreads();
    };
    for (int t = 0; t < count; t += 2 * STAGE) {
        stage(t, 0, in1);
        if (t + STAGE < count) stage(t + STAGE, 1, in0);
    }
    cy.l = row_sum<32>(cy.l);
    if (w0 + col >= r0 + nr) return;
    if (g.n == 1) {
        const float f = failed ? __uint_as_float(0x7FC00000u) : cy.l == 0.0f ? 0.0f : cy.R / cy.l;
        put_out(cy, a, (int64_t)row * a.out_stride + (int64_t)head * a.c.D, gl, f);
    } else {
        const int64_t p = (((int64_t)(seq * a.splits + split) * a.row_tiles + rt) * a.c.H + kvh) * a.rows_cap + 32 * wave + col;
        put_sums(cy, a.part_o + p * a.c.D, gl, cy.R);
        if (gl == 0) reinterpret_cast<float2*>(a.part_ml)[p] = make_float2(cy.m, cy.l);
    }
}

// The row `rr` of n partials, joined and stored, by W = 4 waves of a workgroup or by each wave alone (1).  part(i): number of
// the i-th partial.  A load takes 16 bytes per lane: 64 lanes hold `subs` rows of partials, and eight loads are in flight.
constexpr int FLIGHT = 8;
template <int W, typename F>
__device__ __forceinline__ void join_row(const AttendArgs& a, int n, int rr, int64_t to, int failed, F part) {
    __shared__ float so[4][256], sl[32], sm[32];
    const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, D = a.c.D;
    const int width = D <= 32 ? 8 : D <= 64 ? 16 : D <= 128 ? 32 : 64, subs = 64 / width, sub = lane / width, at = lane % width;
    const bool in = 4 * at < D;
    float m = -__builtin_inff(), l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int b0 = 0; b0 < n; b0 += FLIGHT * W * subs) {
        float2 ml[FLIGHT];
        float4 v[FLIGHT];
#pragma unroll
        for (int u = 0; u < FLIGHT; ++u) {
            const int i = b0 + (u * W + wave) * subs + sub;
            const int64_t p = part(min(i, n - 1)) * a.rows_cap + rr;
            ml[u] = reinterpret_cast<const float2*>(a.part_ml)[p];
            v[u] = *reinterpret_cast<const float4*>(a.part_o + p * D + (in ? 4 * at : 0));
            if (i >= n) ml[u] = make_float2(-__builtin_inff(), 0.0f);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < FLIGHT; ++u) top = fmaxf(top, ml[u].x);
        const float old = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= old;
        o.x *= old, o.y *= old, o.z *= old, o.w *= old;
#pragma unroll
        for (int u = 0; u < FLIGHT; ++u) {
            if (b0 + (u * W + wave) * subs + sub >= n) continue;
            const float f = ml[u].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[u].x - m);
            l = __builtin_fmaf(f, ml[u].y, l);
            o.x = __builtin_fmaf(f, v[u].x, o.x), o.y = __builtin_fmaf(f, v[u].y, o.y);
            o.z = __builtin_fmaf(f, v[u].z, o.z), o.w = __builtin_fmaf(f, v[u].w, o.w);
        }
    }
    if constexpr (W > 1) {
        if (at == 0) sl[wave * subs + sub] = l, sm[wave * subs + sub] = m;
    }
    // the rows of a wave add up in its lanes first
    float top = m;
    for (int w = width; w < 64; w <<= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
    const float f = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    o.x *= f, o.y *= f, o.z *= f, o.w *= f;
    l *= f;
    for (int w = width; w < 64; w <<= 1) {
        o.x += __shfl_xor(o.x, w, 64), o.y += __shfl_xor(o.y, w, 64);
        o.z += __shfl_xor(o.z, w, 64), o.w += __shfl_xor(o.w, w, 64);
        l += __shfl_xor(l, w, 64);
    }
    if constexpr (W == 1) {
        const float z = failed ? __uint_as_float(0x7FC00000u) : l == 0.0f ? 0.0f : 1.0f / l;
        if (sub == 0 && in) store4(a.out, a.type, to + 4 * at, a.out_vec, make_float4(o.x * z, o.y * z, o.z * z, o.w * z));
        return;
    }
    if (sub == 0 && in) *reinterpret_cast<float4*>(&so[wave][4 * at]) = o;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += 256) {
        float most = -__builtin_inff();
        for (int i = 0; i < 4 * subs; ++i) most = fmaxf(most, sm[i]);
        float y = 0.0f, z = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float mw = -__builtin_inff();
            for (int i = 0; i < subs; ++i) {
                const float mi = sm[w * subs + i];
                mw = fmaxf(mw, mi);
                z = __builtin_fmaf(mi == most ? 1.0f : __builtin_amdgcn_exp2f(mi - most), sl[w * subs + i], z);
            }
            y = __builtin_fmaf(mw == most ? 1.0f : __builtin_amdgcn_exp2f(mw - most), so[w][d], y);
        }
        y = z == 0.0f ? 0.0f : y / z;
        if (failed) y = __uint_as_float(0x7FC00000u);
        store1(a.out, a.type, to + d, y);
    }
}

// Rows that k_attend_rows divided: a wave for each row of a row tile, blockIdx.x as there without the splits
__global__ __launch_bounds__(256) void k_attend_join(const AttendArgs a) {
    int item = blockIdx.x;
    const int kvh = item % a.c.H;
    item /= a.c.H;
    const int rt = item % a.row_tiles, seq = item / a.row_tiles;
    const int failed = *a.c.status;
    const KvSeq s = kv_seq(a.c, a.b, seq);
    const int rows = s.n * a.G, r0 = rt * a.tile_rows;
    if (r0 >= rows) return;
    const int nr = min(a.tile_rows, rows - r0);
    const Range g = range_of(a, s, r0, nr);
    if (g.n == 1) return;
    for (int rr = blockIdx.y * 4 + (threadIdx.x >> 6); rr < nr; rr += gridDim.y * 4) {
        const int r = r0 + rr;
        const int64_t to = (int64_t)(s.row0 + r / a.G) * a.out_stride + (int64_t)(kvh * a.G + r % a.G) * a.c.D;
        join_row<1>(a, g.n, rr, to, failed, [&](int i) { return (((int64_t)seq * a.splits + i) * a.row_tiles + rt) * a.c.H + kvh; });
    }
}

// ---------------------------------------------------------------- few rows: the tiles of the whole batch in equal shares

// Every (sequence, kv head) has its tiles one behind the other in one long line, sequences in the batch's order; wave w of
// the launch takes the places w * per .. of the line.  What a wave has of a sequence and head that others share goes to
// LDS; the waves of a workgroup join what belongs together there, and only what workgroups share becomes a partial
// in memory, numbered by the first of the workgroup's waves that has a part: 2 w + 1 where it begins the sequence
// and head, 2 w where it continues one.  (group = 1: every wave's part goes to memory.)
// To begin a sequence and head (its pages, scales and q arrive one behind the other) costs about as much as START tiles:
// 0 / 2 / 4 of them: 62 / 55 / 53 us for 64 sequences of 150 to 8000 tokens (273 MB).
constexpr int START = 4;
struct Line {
    KvSeq s;        // of the lane's sequence (chunk + lane)
    int tiles;      // of its line per head: START and its tiles, none if it has no rows
    uint32_t end;   // places of the chunk's sequences up to this one, all heads
};
__device__ __forceinline__ Line line_of(const AttendArgs& a, int chunk) {
    const int lane = threadIdx.x & 63, i = chunk + lane;
    Line n;
    n.s = KvSeq{0, 0, 0, 0};
    n.tiles = 0;
    if (i < a.b.n_seqs) {
        n.s = kv_seq(a.c, a.b, i);
        if (n.s.n > 0) n.tiles = START + range_of(a, n.s, 0, n.s.n * a.G).tiles;
    }
    n.end = (uint32_t)n.tiles * a.c.H;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = (uint32_t)__shfl_up((int)n.end, o, 64);
        if (lane >= o) n.end += y;
    }
    return n;
}
constexpr int MIN_TILES = 2;  // of a share
// Waves of a SIMD that the registers of k_attend_stream leave room for (and that it is compiled for).  With 16 rows three
// would fit at 128 dimensions, but more loads in flight read slower: 63 us against 50 for 131000 tokens.
__host__ __device__ constexpr int stream_occupancy(int nr, int dt) { return nr == 32 && dt > 4 ? 1 : 2; }
// LDS of a workgroup that joins its waves' parts
inline size_t stream_lds(int rows, int D) { return sizeof(float) * (size_t)8 * rows * (D + 2); }
__device__ __forceinline__ int per_wave(const AttendArgs& a, uint32_t total) {
    return max(MIN_TILES, (int)((total + a.waves - 1) / a.waves));
}

// What a wave left in LDS: a part of a sequence and head (slot 0: continued from the wave before, slot 1: begun)
struct Part {
    int rows, row0, kvh;  // rows 0: none
    bool ends;            // with the last of its tiles
};

template <int NR, int DT, int ND, bool EXT>
__global__ __launch_bounds__(256, stream_occupancy(NR, DT)) void k_attend_stream(const AttendArgs a) {
    extern __shared__ float lds[];  // [4 waves][2 slots][rows_cap][D], then [..][rows_cap][2]
    __shared__ Part parts[4][2];
    __shared__ Line lines[4][64];   // (kept here: the registers are needed for the tiles)
    const int lane = threadIdx.x & 63, gl = lane / NR, col = lane % NR, wave = threadIdx.x >> 6, D = a.c.D;
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave);
    const int failed = *a.c.status;
    float* sums = lds;
    float2* stats = reinterpret_cast<float2*>(lds + (size_t)8 * a.rows_cap * D);
    if (lane < 2) parts[wave][lane].rows = 0;
    uint32_t total, chunk_end;  // places of the line; of the chunk in `lines`
    {
        const Line n = line_of(a, 0);
        lines[wave][lane] = n;
        total = chunk_end = lane_of(n.end, 63);
        for (int c = 64; c < a.b.n_seqs; c += 64) total += lane_of(line_of(a, c).end, 63);
    }
    const int per = per_wave(a, total);
    uint32_t at = (uint32_t)w * per;
    const uint32_t to = min(total, at + per);
    uint32_t base = 0;  // places before the chunk
    int chunk = 0;
    while (at < to) {
        while (at - base >= chunk_end) {
            base += chunk_end;
            chunk += 64;
            const Line n = line_of(a, chunk);
            lines[wave][lane] = n;
            chunk_end = lane_of(n.end, 63);
        }
        const int i = __builtin_ctzll(__ballot(lines[wave][lane].end > at - base));
        const Line& ln = lines[wave][i];
        const KvSeq s = {__builtin_amdgcn_readfirstlane(ln.s.slot), __builtin_amdgcn_readfirstlane(ln.s.len),
                         __builtin_amdgcn_readfirstlane(ln.s.row0), __builtin_amdgcn_readfirstlane(ln.s.n)};
        const int tiles = __builtin_amdgcn_readfirstlane(ln.tiles), rows = s.n * a.G;
        const uint32_t before = at - base - (__builtin_amdgcn_readfirstlane(ln.end) - (uint32_t)tiles * a.c.H);
        const int kvh = before / tiles, p_begin = before - kvh * tiles, share = min((int)(to - at), tiles - p_begin);
        at += share;
        const Range g = range_of(a, s, 0, rows);
        const int t_begin = max(0, p_begin - START), t_end = p_begin + share - START;
        if (t_end < 0 || (t_end == 0 && g.tiles > 0)) continue;  // the next wave begins it
        const int count = t_end - t_begin;  // (none where nothing is visible)
        const int first = g.begin + t_begin;

        const int r = min(col, rows - 1), head = kvh * a.G + r % a.G, row = s.row0 + r / a.G, pos = g.base + r / a.G;
        const int whole_hi = a.causal ? min(s.len, g.base + 1) : s.len;
        const int whole_lo = a.window ? max(0, g.base + s.n - a.window) : 0;
        Carry<NR, DT> cy;
        carry_init(cy);
        attend_tiles<NR, DT, ND, EXT, true>(cy, a, s, kvh, row, head, col < rows, pos, first, 1, count, whole_lo, whole_hi);
        cy.l = row_sum<NR>(cy.l);
        if (count == g.tiles) {
            const float f = failed ? __uint_as_float(0x7FC00000u) : cy.l == 0.0f ? 0.0f : cy.R / cy.l;
            if (col < rows) put_out(cy, a, (int64_t)row * a.out_stride + (int64_t)head * D, gl, f);
        } else {
            const int slot = t_begin == 0;
            const int p = (wave * 2 + slot) * a.rows_cap + col;
            if (a.group == 1) {
                const int64_t q = ((int64_t)w * 2 + slot) * a.rows_cap + col;
                if (col < rows) {
                    put_sums(cy, a.part_o + q * D, gl, cy.R);
                    if (gl == 0) reinterpret_cast<float2*>(a.part_ml)[q] = make_float2(cy.m, cy.l);
                }
                continue;
            }
            if (col < rows) {
                put_sums(cy, sums + (size_t)p * D, gl, cy.R);
                if (gl == 0) stats[p] = make_float2(cy.m, cy.l);
            }
            if (lane == 0) parts[wave][slot] = Part{rows, s.row0, kvh, t_end == g.tiles};
        }
    }
    if (a.group == 1) return;
    __syncthreads();
    // the workgroup's parts: each one that does not continue a part of the wave before, with those that continue it
    for (int f = 0; f < 8; ++f) {
        const int fw = f >> 1, slot = f & 1;
        const Part part = parts[fw][slot];
        if (part.rows == 0 || (slot == 0 && fw > 0)) continue;
        int last = fw;
        bool ends = part.ends;
        while (!ends && last + 1 < 4 && parts[last + 1][0].rows) ends = parts[++last][0].ends;
        const bool whole = slot == 1 && ends;
        for (int i = threadIdx.x; i < part.rows * D; i += 256) {
            const int rr = i / D, d = i - rr * D;
            float m = -__builtin_inff();
            for (int u = fw; u <= last; ++u) m = fmaxf(m, stats[(u * 2 + (u == fw ? slot : 0)) * a.rows_cap + rr].x);
            float o = 0.0f, l = 0.0f;
            for (int u = fw; u <= last; ++u) {
                const int p = (u * 2 + (u == fw ? slot : 0)) * a.rows_cap + rr;
                const float2 ml = stats[p];
                const float e = ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
                l = __builtin_fmaf(e, ml.y, l);
                o = __builtin_fmaf(e, sums[(size_t)p * D + d], o);
            }
            if (whole) {
                float y = l == 0.0f ? 0.0f : o / l;
                if (failed) y = __uint_as_float(0x7FC00000u);
                store1(a.out, a.type, (int64_t)(part.row0 + rr / a.G) * a.out_stride + (int64_t)(part.kvh * a.G + rr % a.G) * D + d, y);
            } else {
                const int64_t p = ((int64_t)(blockIdx.x * 4 + fw) * 2 + slot) * a.rows_cap + rr;
                a.part_o[p * D + d] = o;
                if (d == 0) reinterpret_cast<float2*>(a.part_ml)[p] = make_float2(m, l);
            }
        }
    }
}

// blockIdx.x = sequence * H + kv head; the rows over blockIdx.y
__global__ __launch_bounds__(256) void k_attend_stream_join(const AttendArgs a) {
    const int seq = blockIdx.x / a.c.H, kvh = blockIdx.x % a.c.H;
    const int failed = *a.c.status;
    uint32_t total = 0, begin = 0;
    KvSeq s = {0, 0, 0, 0};
    int tiles = 0;
    for (int c = 0; c < a.b.n_seqs; c += 64) {
        const Line n = line_of(a, c);
        if (c == (seq & ~63)) {
            const int i = seq & 63;
            s = KvSeq{lane_of(n.s.slot, i), lane_of(n.s.len, i), lane_of(n.s.row0, i), lane_of(n.s.n, i)};
            tiles = lane_of(n.tiles, i);
            begin = total + lane_of(n.end, i) - (uint32_t)tiles * (a.c.H - kvh);
        }
        total += lane_of(n.end, 63);
    }
    const int rows = s.n * a.G, per = per_wave(a, total);
    if (tiles <= START) return;
    const int w0 = (begin + START) / per, b0 = w0 / a.group, b1 = (int)((begin + tiles - 1) / per) / a.group;
    if (b0 == b1) return;
    auto part = [&](int i) { return i == 0 ? (int64_t)w0 * 2 + 1 : (int64_t)(b0 + i) * a.group * 2; };
    auto place = [&](int r) { return (int64_t)(s.row0 + r / a.G) * a.out_stride + (int64_t)(kvh * a.G + r % a.G) * a.c.D; };
    if (b1 - b0 < 2 * FLIGHT) {  // few partials: a wave for each row
        for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.y * 4) join_row<1>(a, b1 - b0 + 1, r, place(r), failed, part);
        return;
    }
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        join_row<4>(a, b1 - b0 + 1, r, place(r), failed, part);
        __syncthreads();
    }
}

template <typename K>
void launch_k(K k, unsigned grid, int threads, size_t lds, const AttendArgs& a, hipStream_t st) {
    if (lds > 48 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(k, dim3(grid), dim3(threads), lds, st, a);
}
#define JX_ATTEND_FORM(kernel, ...)                                                       \
    (wide ? (ext ? kernel<__VA_ARGS__, 3, true> : kernel<__VA_ARGS__, 3, false>)          \
          : (ext ? kernel<__VA_ARGS__, 2, true> : kernel<__VA_ARGS__, 2, false>))

template <int NR, int DT>
void launch_form(const AttendArgs& a, bool ext, bool wide, hipStream_t st) {
    if (a.waves)
        launch_k(JX_ATTEND_FORM(k_attend_stream, NR, DT), a.waves / 4, 256, a.group == 1 ? 0 : stream_lds(a.rows_cap, a.c.D), a, st);
    else
        launch_k(JX_ATTEND_FORM(k_attend, NR, DT), (unsigned)(a.b.n_seqs * a.c.H), 64 * waves_of(DT),
                 sizeof(float) * (size_t)waves_of(DT) * a.rows_cap * (a.c.D + 2), a, st);
}
template <int DT>
void launch_dt(const AttendArgs& a, hipStream_t st) {
    const bool ext = a.cap > 0.0f || a.alibi, wide = a.type == JX_TYPE_F32;
    if (a.tile_rows > 32)
        launch_k(JX_ATTEND_FORM(k_attend_rows, DT), (unsigned)((int64_t)a.b.n_seqs * a.splits * a.row_tiles * a.c.H), 64 * ROWS_W,
                 (size_t)2 * STAGE * 4096 * DT, a, st);
    else if (a.rows_cap <= 16)
        launch_form<16, DT>(a, ext, wide, st);
    else
        launch_form<32, DT>(a, ext, wide, st);
}

}  // namespace

AttendPlan attend_plan(const jx_kv_cache& c, const jx_kv_batch& b, const jx_attention& t) {
    AttendPlan p;
    const int64_t most = (int64_t)c.max_pages * c.page_tokens;
    const int G = t.n_heads / c.n_kv_heads, DT = c.head_dim / 32, W = waves_of(DT);
    const int64_t rows = (int64_t)b.max_rows * G;
    int64_t len = b.max_len > 0 ? std::min<int64_t>(b.max_len, most) : most;
    if (t.window > 0 && t.causal) len = std::min<int64_t>(len, (int64_t)t.window + b.max_rows + KV_BLOCK);
    const int64_t tiles = std::max<int64_t>(1, (len + KV_BLOCK - 1) / KV_BLOCK);
    // a line of the batch's tiles has its places in 32 bits
    const bool line = (int64_t)b.n_seqs * c.n_kv_heads * ((most + KV_BLOCK - 1) / KV_BLOCK + START) < INT32_MAX;
    p.splits = 1;
    p.chunk = (int)tiles;
    p.waves = 0;
    p.group = 1;
    p.partials = 0;
    if (rows <= 32 && line) {
        const int64_t items = (int64_t)b.n_seqs * c.n_kv_heads;
        p.tile_rows = 32;
        p.row_tiles = 1;
        p.rows_cap = (int)rows;
        if (items <= 256 && tiles <= 4 * W) return p;  // a workgroup for each sequence and kv head, four tiles per wave at most
        // few sequences and heads have many parts each: 8 of them 57 us with a group's parts joined and 58 without, 64 (draft
        // tokens, 10 rows of 256 dimensions) 32 and 33; 272 and 512 of them 22 and 21, 60 and 58
        const size_t lds = stream_lds(p.rows_cap, c.head_dim);
        p.group = items <= 128 && lds <= 150 * 1024 ? 4 : 1;
        // as many waves as are resident at once: registers, and 160 KB of LDS less the workgroup's fixed 7
        p.waves = 256 * 4 * (p.group == 4 && lds > 72 * 1024 ? 1 : stream_occupancy(rows <= 16 ? 16 : 32, DT));
        p.partials = 2 * (int64_t)p.waves;
        return p;
    }
    p.tile_rows = 32 * ROWS_W;
    p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    p.rows_cap = (int)std::min<int64_t>(p.tile_rows, rows);
    const int64_t items = (int64_t)b.n_seqs * p.row_tiles * c.n_kv_heads;
    // Two workgroups share a CU, and sequences of several lengths need more to even out: up to 2048 of at least 16 tiles.  Five
    // pieces of prompts (440 workgroups undivided): 113 us undivided, 70 in two parts, 50 in five, and the join
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(2048 / std::max<int64_t>(1, items), tiles / 16));
    p.chunk = (int)((tiles + splits - 1) / splits);
    p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
    if (p.splits > 1) p.partials = items * p.splits;
    return p;
}

void launch_attend(const AttendArgs& a, hipStream_t st) {
    switch (a.c.D / 32) {
        case 1: launch_dt<1>(a, st); break;
        case 2: launch_dt<2>(a, st); break;
        case 3: launch_dt<3>(a, st); break;
        case 4: launch_dt<4>(a, st); break;
        case 5: launch_dt<5>(a, st); break;
        case 6: launch_dt<6>(a, st); break;
        case 7: launch_dt<7>(a, st); break;
        default: launch_dt<8>(a, st); break;
    }
    const unsigned pairs = (unsigned)(a.b.n_seqs * a.c.H);
    if (a.waves)  // few sequences and heads: a workgroup per row (many partials each); many: one for all rows
        hipLaunchKernelGGL(k_attend_stream_join, dim3(pairs, pairs <= 128 ? a.rows_cap : 1), dim3(256), 0, st, a);
    else if (a.splits > 1)
        hipLaunchKernelGGL(k_attend_join, dim3(pairs * a.row_tiles, (a.rows_cap + 31) / 32), dim3(256), 0, st, a);
}

}  // namespace jx
