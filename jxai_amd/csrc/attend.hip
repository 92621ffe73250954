// Attention of query rows over the paged 8-bit cache.
//
// A wave takes 32 rows of one sequence and kv head (row = token of the call, head within the group) against a block of 32
// tokens at a time, everything in registers:
//   S^T = K Q^T   32x32x32 int8 MFMAs: the codes of K as they lie in memory (one 16-byte load per lane and 32 dimensions)
//                 against q as two (fp32: three) signed digits of 7 bits, exact in int32
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

// ND signed digits of q in MFMA operand order: lane (h, c) holds dimensions 32 j + 16 h .. + 15 of row c.  qs: the value of
// one unit of the last digit, NaN where the row has a value that is not finite.
template <int DT, int ND>
__device__ __forceinline__ void load_q(const AttendArgs& a, int row, int head, int h, bool valid, v4i (&qd)[ND][DT], float& qs) {
    constexpr float TOP = ND == 2 ? 127.0f * 128.0f : 127.0f * 16384.0f;
    float v[DT][16];
    uint32_t top = 0;
    const int64_t at = (int64_t)row * a.q_stride + (int64_t)head * a.c.D + 16 * h;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
        if (valid) {
            load16(a.q, a.type, at + 32 * j, a.q_vec, v[j]);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[j][k] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(v[j][k]) & 0x7FFFFFFFu);  // orders NaN and infinity last
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    const bool finite = top < 0x7F800000u;
    // rows below 2^-100 count as zero: TOP / amax stays finite
    const bool zero = top < 0x0D800000u;
    const float amax = __uint_as_float(top);
    const float inv = finite && !zero ? TOP / amax : 0.0f;
    qs = !finite ? __uint_as_float(0x7FC00000u) : zero ? 0.0f : amax / TOP;
#pragma unroll
    for (int j = 0; j < DT; ++j) {
        uint32_t w[ND][4] = {};
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            int u = finite ? (int)__builtin_rintf(v[j][k] * inv) : 0;
#pragma unroll
            for (int n = ND - 1; n > 0; --n) {  // last digits first, -64 .. 63
                const int up = (u + 64) >> 7;
                w[n][k >> 2] |= (uint32_t)((u - (up << 7)) & 255) << (8 * (k & 3));
                u = up;
            }
            w[0][k >> 2] |= (uint32_t)(u & 255) << (8 * (k & 3));
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) qd[n][j] = v4i{(int)w[n][0], (int)w[n][1], (int)w[n][2], (int)w[n][3]};
    }
}

// What a wave carries for its 32 rows.
template <int DT>
struct Carry {
    v16f o[DT];
    float m, l;  // of the lane's row: reference maximum (log2), sum of the weights of this lane half
    float R;     // largest scale of V's blocks so far
};

template <int DT>
__device__ __forceinline__ void carry_init(Carry<DT>& s) {
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) s.o[i][k] = 0.0f;
    s.m = -__builtin_inff();
    s.l = 0.0f;
    s.R = 0.0f;
}

template <int DT>
__device__ __forceinline__ void carry_scale(Carry<DT>& s, float f) {
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) s.o[i][k] *= f;
}

__device__ __forceinline__ h8 codes_to_half(uint32_t w0, uint32_t w1) {
    const h2v one = {(_Float16)1.0f, (_Float16)1.0f}, bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return cvt8(w0, w1, 0xFFFFFFFFu, 0x80808080u, one, bias);  // 1024 + (code + 128) - 1152
}

// One block of 32 tokens from t0 on.  lo / hi: the lane's row sees tokens lo .. hi - 1 (masked: whether to look).
template <int DT, int ND, bool EXT>
__device__ __forceinline__ void tile(Carry<DT>& s, const AttendArgs& a, const v4i (&qd)[ND][DT], float qs, float slope, int pos,
                                     const v4i (&kc)[DT], const v4i (&vc)[DT], float ks, float vs, int t0, int h, int lo, int hi,
                                     bool masked) {
    v16i acc[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n) {
        acc[n] = v16i{};
#pragma unroll
        for (int j = 0; j < DT; ++j) acc[n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(kc[j], qd[n][j], acc[n], 0, 0, 0);
    }
    float x[16];
    const float c = qs * ks * (EXT ? a.scale : a.scale2);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        // |acc| <= 127 * 127 * 256: two digits fit an int32
        if constexpr (ND == 2)
            x[i] = (float)(acc[0][i] * 128 + acc[1][i]) * c;
        else
            x[i] = __builtin_fmaf((float)acc[0][i], 16384.0f, (float)(acc[1][i] * 128 + acc[2][i])) * c;
    }
    if constexpr (EXT) {
        if (a.cap > 0.0f) {
            const float inv = 1.0f / a.cap;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = a.cap * tanh_fast(x[i] * inv);
        }
        const float d0 = (float)(t0 + 4 * h - pos);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(slope, d0 + (float)(8 * (i >> 2) + (i & 3)), x[i]) * LOG2E;
    }
    if (masked) {
        const int l0 = lo - t0 - 4 * h, h0 = hi - t0 - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = 8 * (i >> 2) + (i & 3);
            x[i] = t >= l0 && t < h0 ? x[i] : -__builtin_inff();
        }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > s.m + LAG)) {
        const float m = fmaxf(s.m, top);
        const float f = m == s.m ? 1.0f : __builtin_amdgcn_exp2f(s.m - m);
        s.m = m;
        s.l *= f;
        carry_scale(s, f);
    }
    if (vs > s.R) {
        carry_scale(s, s.R / vs);
        s.R = vs;
    }
    // a block of zeros has scale 0; NaN marks a block that reads as NaN
    const float vr = vs == s.R && vs > 0.0f ? 1.0f : vs == 0.0f ? 0.0f : vs / s.R;
    const float ref = s.m == -__builtin_inff() ? (float)-OFF : s.m - (float)OFF;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(x[i] - ref);
        sum += p;
        x[i] = p * vr;
    }
    if (masked) {  // nothing of a NaN scale reaches a row that does not see the block
        const int l0 = lo - t0 - 4 * h, h0 = hi - t0 - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = 8 * (i >> 2) + (i & 3);
            x[i] = t >= l0 && t < h0 ? x[i] : 0.0f;
        }
    }
    s.l += sum;
    // token 8 a + 4 h + b is register 4 a + b here and byte 8 (a & 1) + 4 (a >> 1) + b of V
    h8 p0, p1, e0, e1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p0[i] = (_Float16)x[i], p0[4 + i] = (_Float16)x[8 + i];
        p1[i] = (_Float16)x[4 + i], p1[4 + i] = (_Float16)x[12 + i];
    }
    if constexpr (ND == 3) {  // the weights' remainders: 22 bits in all
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e0[i] = (_Float16)(x[i] - (float)p0[i]), e0[4 + i] = (_Float16)(x[8 + i] - (float)p0[4 + i]);
            e1[i] = (_Float16)(x[4 + i] - (float)p1[i]), e1[4 + i] = (_Float16)(x[12 + i] - (float)p1[4 + i]);
        }
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
        const h8 v0 = codes_to_half((uint32_t)vc[i][0], (uint32_t)vc[i][1]);
        const h8 v1 = codes_to_half((uint32_t)vc[i][2], (uint32_t)vc[i][3]);
        s.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, p0, s.o[i], 0, 0, 0);
        s.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, p1, s.o[i], 0, 0, 0);
        if constexpr (ND == 3) {
            s.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, e0, s.o[i], 0, 0, 0);
            s.o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, e1, s.o[i], 0, 0, 0);
        }
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

// blockIdx.x = ((sequence * splits + split) * row_tiles + row tile) * H + kv head.  The waves of a workgroup take the tiles of
// its split in turn and join in LDS.
template <int DT, int ND, bool EXT>
__global__ __launch_bounds__(64 * waves_of(DT)) void k_attend(const AttendArgs a) {
    extern __shared__ float lds[];
    const int W = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    int item = blockIdx.x;
    const int kvh = item % a.c.H;
    item /= a.c.H;
    const int rt = item % a.row_tiles;
    item /= a.row_tiles;
    const int split = item % a.splits, seq = item / a.splits;
    const int failed = *a.c.status;
    const KvSeq s = kv_seq(a.c, a.b, seq);
    const int rows = s.n * a.G, r0 = rt * 32;
    if (r0 >= rows) return;
    const int nr = min(32, rows - r0);
    const Range g = range_of(a, s, r0, nr);
    if (split >= g.n) return;
    const int r = r0 + min(col, nr - 1), head = kvh * a.G + r % a.G, row = s.row0 + r / a.G, pos = g.base + r / a.G;
    const int hi = a.causal ? min(s.len, pos + 1) : s.len, lo = a.window ? max(0, pos - a.window + 1) : 0;
    // tiles that every row sees whole need no mask: hi of the first row, lo of the last
    const int p0 = g.base + r0 / a.G, p1 = g.base + (r0 + nr - 1) / a.G;
    const int whole_hi = a.causal ? min(s.len, p0 + 1) : s.len, whole_lo = a.window ? max(0, p1 - a.window + 1) : 0;

    v4i qd[ND][DT];
    float qs;
    load_q<DT, ND>(a, row, head, h, col < nr, qd, qs);
    const float slope = EXT && a.alibi ? a.alibi[head] : 0.0f;
    Carry<DT> cy;
    carry_init(cy);

    const int first = g.begin + split * g.per + wave, end = g.begin + min(g.tiles, (split + 1) * g.per);
    const int mine = first < end ? (end - first + W - 1) / W : 0;
    const int64_t bytes = (int64_t)KV_BLOCK * a.c.D;
    for (int b0 = 0; b0 < mine; b0 += 64) {
        // the lane's tile of the next 64: its blocks and scales
        int kb = 0, vb = 0;
        float ks = 0.0f, vs = 0.0f;
        if (b0 + lane < mine) {
            const int t = first + (b0 + lane) * W;
            int page = a.c.table[(int64_t)s.slot * a.c.max_pages + (t >> a.c.blocks_shift)];
            const bool bad = page < 0 || page >= a.c.n_pages;
            page = bad ? 0 : page;
            const int blk = t & ((1 << a.c.blocks_shift) - 1);
            kb = a.c.block_index(page, 0, kvh, blk);
            vb = a.c.block_index(page, 1, kvh, blk);
            ks = a.c.scales[kb];
            vs = a.c.scales[vb];
            if (bad) {
                ks = vs = __uint_as_float(0x7FC00000u);
                atomicOr(a.c.status, JX_KV_BAD_PAGE);
            }
        }
        const int count = min(64, mine - b0);
        v4i kc[DT], vc[DT], kn[DT], vn[DT];
        auto fetch = [&](int i, v4i(&k)[DT], v4i(&v)[DT]) {
            const int8_t* kp = a.c.codes + __builtin_amdgcn_readlane(kb, i) * bytes + lane * 16;
            const int8_t* vp = a.c.codes + __builtin_amdgcn_readlane(vb, i) * bytes + h * (16 * a.c.D) + col * 16;
#pragma unroll
            for (int j = 0; j < DT; ++j) k[j] = *reinterpret_cast<const v4i*>(kp + j * 1024);
#pragma unroll
            for (int j = 0; j < DT; ++j) v[j] = *reinterpret_cast<const v4i*>(vp + j * 512);
        };
        fetch(0, kc, vc);
        for (int i = 0; i < count; ++i) {
            if (i + 1 < count) fetch(i + 1, kn, vn);
            const int t0 = (first + (b0 + i) * W) * KV_BLOCK;
            const float ki = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), i));
            const float vi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), i));
            tile<DT, ND, EXT>(cy, a, qd, qs, slope, pos, kc, vc, ki, vi, t0, h, lo, hi, t0 < whole_lo || t0 + KV_BLOCK > whole_hi);
#pragma unroll
            for (int j = 0; j < DT; ++j) kc[j] = kn[j], vc[j] = vn[j];
        }
    }

    // the waves' sums: [W][rows_cap][D], then [W][rows_cap][2] with the maximum and the sum of weights
    float* so = lds;
    float* sm = lds + (size_t)W * a.rows_cap * a.c.D;
    cy.l += __shfl_xor(cy.l, 32, 64);
    if (col < nr) {
        float* o = so + ((size_t)wave * a.rows_cap + col) * a.c.D;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float4*>(o + 32 * i + 8 * k + 4 * h) =
                    make_float4(cy.o[i][4 * k] * cy.R, cy.o[i][4 * k + 1] * cy.R, cy.o[i][4 * k + 2] * cy.R, cy.o[i][4 * k + 3] * cy.R);
        if (h == 0) {
            sm[(wave * a.rows_cap + col) * 2] = cy.m;
            sm[(wave * a.rows_cap + col) * 2 + 1] = cy.l;
        }
    }
    __syncthreads();
    const int D = a.c.D;
    for (int i = threadIdx.x; i < nr * D; i += blockDim.x) {
        const int rr = i / D, d = i - rr * D;
        float m = -__builtin_inff();
        for (int w = 0; w < W; ++w) m = fmaxf(m, sm[(w * a.rows_cap + rr) * 2]);
        float o = 0.0f, l = 0.0f;
        for (int w = 0; w < W; ++w) {
            const float mw = sm[(w * a.rows_cap + rr) * 2];
            const float f = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
            l = __builtin_fmaf(f, sm[(w * a.rows_cap + rr) * 2 + 1], l);
            o = __builtin_fmaf(f, so[((size_t)w * a.rows_cap + rr) * D + d], o);
        }
        const int orow = s.row0 + (r0 + rr) / a.G, ohead = kvh * a.G + (r0 + rr) % a.G;
        if (g.n == 1) {
            float y = l == 0.0f ? 0.0f : o / l;
            if (failed) y = __uint_as_float(0x7FC00000u);
            store1(a.out, a.type, (int64_t)orow * a.out_stride + (int64_t)ohead * D + d, y);
        } else {
            const int64_t at = ((int64_t)orow * a.heads + ohead) * a.splits + split;
            a.part_o[at * D + d] = o;
            if (d == 0) a.part_ml[at * 2] = m, a.part_ml[at * 2 + 1] = l;
        }
    }
}

// Rows that were divided: their splits' sums joined.  A wave per row; grid as k_attend's without the splits.
__global__ __launch_bounds__(256) void k_attend_join(const AttendArgs a) {
    int item = blockIdx.x;
    const int kvh = item % a.c.H;
    item /= a.c.H;
    const int rt = item % a.row_tiles, seq = item / a.row_tiles;
    const int failed = *a.c.status;
    const KvSeq s = kv_seq(a.c, a.b, seq);
    const int rows = s.n * a.G, r0 = rt * 32;
    if (r0 >= rows) return;
    const int nr = min(32, rows - r0);
    const Range g = range_of(a, s, r0, nr);
    if (g.n == 1) return;
    const int lane = threadIdx.x & 63, D = a.c.D;
    for (int rr = threadIdx.x >> 6; rr < nr; rr += blockDim.x >> 6) {
        const int row = s.row0 + (r0 + rr) / a.G, head = kvh * a.G + (r0 + rr) % a.G;
        const int64_t at = ((int64_t)row * a.heads + head) * a.splits;
        float m = -__builtin_inff();
        for (int i = 0; i < g.n; ++i) m = fmaxf(m, a.part_ml[(at + i) * 2]);
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
        for (int i = 0; i < g.n; ++i) {
            const float mi = a.part_ml[(at + i) * 2];
            const float f = mi == m ? 1.0f : __builtin_amdgcn_exp2f(mi - m);
            l = __builtin_fmaf(f, a.part_ml[(at + i) * 2 + 1], l);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (lane + 64 * k < D) o[k] = __builtin_fmaf(f, a.part_o[(at + i) * D + lane + 64 * k], o[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < D) {
                float y = l == 0.0f ? 0.0f : o[k] / l;
                if (failed) y = __uint_as_float(0x7FC00000u);
                store1(a.out, a.type, (int64_t)row * a.out_stride + (int64_t)head * D + lane + 64 * k, y);
            }
    }
}

template <int DT>
void launch_dt(const AttendArgs& a, hipStream_t st) {
    const size_t lds = sizeof(float) * (size_t)waves_of(DT) * a.rows_cap * (a.c.D + 2);
    const dim3 grid((unsigned)((int64_t)a.b.n_seqs * a.splits * a.row_tiles * a.c.H));
    const bool ext = a.cap > 0.0f || a.alibi, wide = a.type == JX_TYPE_F32;
    auto k = wide ? (ext ? k_attend<DT, 3, true> : k_attend<DT, 3, false>) : (ext ? k_attend<DT, 2, true> : k_attend<DT, 2, false>);
    if (lds > 65536)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(k, grid, dim3(64 * waves_of(DT)), lds, st, a);
}

}  // namespace

AttendPlan attend_plan(const jx_kv_cache& c, const jx_kv_batch& b, const jx_attention& t) {
    AttendPlan p;
    const int64_t most = (int64_t)c.max_pages * c.page_tokens;
    const int G = t.n_heads / c.n_kv_heads;
    p.row_tiles = (int)(((int64_t)b.max_rows * G + 31) / 32);
    int64_t len = b.max_len > 0 ? std::min<int64_t>(b.max_len, most) : most;
    if (t.window > 0 && t.causal) len = std::min<int64_t>(len, (int64_t)t.window + b.max_rows + KV_BLOCK);
    const int64_t tiles = std::max<int64_t>(1, (len + KV_BLOCK - 1) / KV_BLOCK);
    // about two workgroups for each of the 256 CUs, of at least two tiles per wave
    const int64_t items = (int64_t)b.n_seqs * p.row_tiles * c.n_kv_heads;
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(1, items), tiles / (2 * waves_of(c.head_dim / 32))));
    p.chunk = (int)((tiles + splits - 1) / splits);
    p.splits = (int)((tiles + p.chunk - 1) / p.chunk);
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
    if (a.splits > 1)
        hipLaunchKernelGGL(k_attend_join, dim3((unsigned)((int64_t)a.b.n_seqs * a.row_tiles * a.c.H)), dim3(256), 0, st, a);
}

}  // namespace jx
