// The paged 8-bit key/value cache: new tokens into it, its pages (reserve, trim, fork, compact), and the C entry points of the
// cache and its attention.
#include <algorithm>
#include <cmath>

#include "jxmoe_device.h"
#include "jxmoe_kv.h"

namespace jx {
namespace {

constexpr float TINY = 7.52316384526264e-37f;  // 2^-120: smaller scales are zero, so that 1 / scale is finite
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7FC00000u); }

// ---------------------------------------------------------------- append

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<_Float16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float widen<__bf16>(__bf16 v) { return (float)v; }

// The integer nearest to v / s (ties to the even one), |v| at most 127 s and a rounding: inv = 1 / s, half = s / 2.  The
// product's rounding can miss by one next to the middle of two integers, so the remainder decides: v - q s is a
// multiple of half an ulp of s and below 2 s, hence exact from one fused multiply-add where it is near s / 2.
__device__ __forceinline__ int nearest(float v, float s, float inv, float half) {
    float q = __builtin_rintf(v * inv);
    const float e = __builtin_fmaf(-q, s, v), ae = __builtin_fabsf(e);
    if (ae > half || (ae == half && ((int)q & 1))) q += __builtin_copysignf(1.0f, e);
    return (int)q;
}

struct AppendArgs {
    KvView c;
    KvRows b;
    const int32_t* ref;
    const void *k, *v;
    int64_t stride;
    int blocks;  // of a sequence's rows at most
    bool vec;    // rows aligned to 16 bytes
};

// N consecutive values; vec: aligned to N of them (or to 16 bytes)
template <typename T, int N>
__device__ __forceinline__ void load_values(const T* p, bool vec, float* v) {
    if (vec) {
        typedef T V __attribute__((ext_vector_type(N * sizeof(T) > 16 ? 16 / sizeof(T) : N)));
        constexpr int M = sizeof(V) / sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += M) {
            const V u = *reinterpret_cast<const V*>(p + i);
#pragma unroll
            for (int k = 0; k < M; ++k) v[i + k] = widen<T>(u[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = widen<T>(p[k]);
    }
}

// The block's scale after the new tokens (top: bits of their largest magnitude) and, if it grew, `grew`.
__device__ __forceinline__ float new_scale(uint32_t top, float before, bool& grew) {
    const float amax = __uint_as_float(top);
    float s = amax / 127.0f;
    s = s < TINY ? 0.0f : s;
    if (top >= 0x7F800000u || before != before) {
        grew = false;
        return quiet_nan();
    }
    grew = s > before;
    return grew ? s : before;
}

// An earlier code at its block's new scale: the integer nearest to code * before / now.  Both products have 31 bits, so their
// difference in 64 bits is exact.
__device__ __forceinline__ int recode(int code, float before, float now, float ratio) {
    float q = __builtin_rintf((float)code * ratio);
    const double e = (double)code * (double)before - (double)q * (double)now, ae = __builtin_fabs(e), half = 0.5 * (double)now;
    if (ae > half || (ae == half && ((int)q & 1))) q += __builtin_copysignf(1.0f, (float)e);
    return (int)q;
}
__device__ __forceinline__ uint32_t recode4(uint32_t w, float before, float now) {
    const float ratio = before / now;
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) r |= (uint32_t)(recode((int)(int8_t)(w >> (8 * k)), before, now, ratio) & 255) << (8 * k);
    return r;
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

// One wave for one block of 32 tokens of a kv head, K (blockIdx.z = 0) or V.  Bound by HBM for prompts (each lane's loads and
// stores are 8 to 64 bytes in a row: 33.5 MB in and 16.8 out take 20 us), by the chain status, length, page, value, code
// for single tokens, whose codes are written byte by byte without reading the block.
template <typename T, int DT>
__global__ __launch_bounds__(64) void k_append(const AppendArgs a) {
    if (*a.c.status) return;
    const int lane = threadIdx.x, h = lane >> 5, r = lane & 31;
    const KvSeq s = kv_seq(a.c, a.b, blockIdx.x / a.blocks);
    const int begin = s.len - s.n;
    if (s.n == 0) return;
    if (begin < 0) {  // more rows than tokens
        if (lane == 0) atomicOr(a.c.status, JX_KV_BAD_ARG);
        return;
    }
    const int block = begin / KV_BLOCK + blockIdx.x % a.blocks, t0 = block * KV_BLOCK;
    if (t0 >= s.len) return;
    const int page = a.c.table[(int64_t)s.slot * a.c.max_pages + (block >> a.c.blocks_shift)];
    if (page < 0 || page >= a.c.n_pages) {
        if (lane == 0) atomicOr(a.c.status, JX_KV_BAD_PAGE);
        return;
    }
    if (a.ref[page] > 1) {  // another sequence reads this page
        if (lane == 0) atomicOr(a.c.status, JX_KV_SHARED);
        return;
    }
    const int head = blockIdx.y, which = blockIdx.z;
    const int index = a.c.block_index(page, which, head, block & ((1 << a.c.blocks_shift) - 1));
    int8_t* codes = a.c.codes + (int64_t)index * (KV_BLOCK * a.c.D);
    const float before = t0 < begin ? a.c.scales[index] : 0.0f;
    const T* x = reinterpret_cast<const T*>(which ? a.v : a.k) + (int64_t)head * a.c.D + (int64_t)(s.row0 - begin) * a.stride;
    bool grew;
    uint32_t top = 0;
    auto code = [&](float v, float now, float inv, float half) { return (uint32_t)((inv > 0.0f ? nearest(v, now, inv, half) : 0) & 255); };
    const int lo = max(begin, t0), hi = min(s.len, t0 + KV_BLOCK);  // the new tokens
    // the block's earlier codes at a scale that grew: K's rows below lo, V's bytes
    auto recode_k = [&](float now) {
        uint4* at = reinterpret_cast<uint4*>(codes) + h * 32 + r;
        if (t0 + r < lo)
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                const uint4 u = at[j * 64];
                at[j * 64] = make_uint4(recode4(u.x, before, now), recode4(u.y, before, now), recode4(u.z, before, now), recode4(u.w, before, now));
            }
    };
    auto token_of = [&](int k) { return t0 + 8 * (2 * ((k >> 2) & 1) + (k >> 3)) + 4 * h + (k & 3); };  // of byte k of the lane half's pieces
    if (hi - lo == 1) {
        // one new token: the lane's values lane + 64 i
        constexpr int N = (DT + 1) / 2;
        float v[N];
        const T* row = x + (int64_t)lo * a.stride;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = lane + 64 * i < 32 * DT ? widen<T>(row[lane + 64 * i]) : 0.0f;
            top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        }
        const float now = new_scale(wave_umax(top), before, grew);
        const float inv = now > 0.0f ? 1.0f / now : 0.0f, half = 0.5f * now;
        if (lane == 0) a.c.scales[index] = now;
        if (grew && lo > t0) {
            if (which == 0) {
                recode_k(now);
            } else {
                uint4* at = reinterpret_cast<uint4*>(codes) + h * 32 * DT + r;
                uint32_t keep[4] = {};
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (token_of(k) < lo) keep[k >> 2] |= 255u << (8 * (k & 3));
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    const uint4 u = at[j * 32];
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[k] = keep[k] ? (recode4(w[k], before, now) & keep[k]) | (w[k] & ~keep[k]) : w[k];
                    at[j * 32] = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            // the new token's bytes lie in words that other lanes have just stored whole
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const int t = lo - t0, ta = t >> 3, th = (t >> 2) & 1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = lane + 64 * i;
            if (d >= 32 * DT) break;
            const int at = which == 0 ? (d >> 4) * 512 + t * 16 + (d & 15) : (th * 32 * DT + d) * 16 + 8 * (ta & 1) + 4 * (ta >> 1) + (t & 3);
            codes[at] = (int8_t)code(v[i], now, inv, half);
        }
        return;
    }
    if (which == 0) {
        // lane (h, r): dimensions 32 j + 16 h .. + 15 of token r
        const bool fresh = t0 + r >= lo && t0 + r < hi;
        float v[DT][16];
        // (lanes without a new token read the nearest one, which changes no maximum: all loads are in flight together)
        const T* row = x + (int64_t)min(max(t0 + r, lo), hi - 1) * a.stride + 16 * h;
#pragma unroll
        for (int j = 0; j < DT; ++j) load_values<T, 16>(row + 32 * j, a.vec, v[j]);
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(v[j][k]) & 0x7FFFFFFFu);
        const float now = new_scale(wave_umax(top), before, grew);
        const float inv = now > 0.0f ? 1.0f / now : 0.0f, half = 0.5f * now;
        if (lane == 0) a.c.scales[index] = now;
        uint4* to = reinterpret_cast<uint4*>(codes) + h * 32 + r;
        if (fresh) {
#pragma unroll
            for (int j = 0; j < DT; ++j) {
                uint32_t w[4] = {};
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k >> 2] |= code(v[j][k], now, inv, half) << (8 * (k & 3));
                to[j * 64] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else if (grew) {
            recode_k(now);
        }
    } else {
        // lane (h, r): dimensions 128 j + 4 r .. + 3 of the 16 tokens 8 a + 4 h + b, four pieces of 16 bytes in a row
        constexpr int N = (DT + 3) / 4;
        float v[N][16][4];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int d = 128 * j + 4 * r < 32 * DT ? 128 * j + 4 * r : 4 * r;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                load_values<T, 4>(x + (int64_t)min(max(token_of(k), lo), hi - 1) * a.stride + (d < 32 * DT ? d : 0), a.vec, v[j][k]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[j][k][i]) & 0x7FFFFFFFu);
        const float now = new_scale(wave_umax(top), before, grew);
        const float inv = now > 0.0f ? 1.0f / now : 0.0f, half = 0.5f * now;
        if (lane == 0) a.c.scales[index] = now;
        uint32_t keep[4] = {}, put[4] = {};  // bytes of earlier tokens, of new tokens
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int t = token_of(k);
            if (t < lo) keep[k >> 2] |= 255u << (8 * (k & 3));
            if (t >= lo && t < hi) put[k >> 2] |= 255u << (8 * (k & 3));
        }
        const bool whole = (put[0] & put[1] & put[2] & put[3]) == 0xFFFFFFFFu;
        const bool some = (put[0] | put[1] | put[2] | put[3]) != 0 || grew;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int d = 128 * j + 4 * r;
            if (d >= 32 * DT || !some) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4* to = reinterpret_cast<uint4*>(codes) + h * 32 * DT + d + i;
                uint32_t w[4] = {};
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k >> 2] |= code(v[j][k][i], now, inv, half) << (8 * (k & 3));
                if (!whole) {
                    const uint4 u4 = *to;
                    const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t old = grew && keep[k] ? recode4(u[k], before, now) : u[k];
                        w[k] = (w[k] & put[k]) | (old & keep[k]) | (u[k] & ~(put[k] | keep[k]));
                    }
                }
                *to = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

template <typename T>
void append_type(const AppendArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.b.n_seqs * a.blocks), (unsigned)a.c.H, 2);
    auto k = k_append<T, 8>;
    switch (a.c.D / 32) {
        case 1: k = k_append<T, 1>; break;
        case 2: k = k_append<T, 2>; break;
        case 3: k = k_append<T, 3>; break;
        case 4: k = k_append<T, 4>; break;
        case 5: k = k_append<T, 5>; break;
        case 6: k = k_append<T, 6>; break;
        case 7: k = k_append<T, 7>; break;
        default: break;
    }
    hipLaunchKernelGGL(k, grid, dim3(64), 0, st, a);
}

// ---------------------------------------------------------------- pages

// Sections of the scratch memory
struct Book {
    int32_t* head;   // [0] copies, [1] pages in use before a compaction's moves
    int32_t *from, *to;   // [max(n_pages, max_seqs)] the copies
    int32_t* remap;  // [n_pages] new place of a moved page
    int32_t* fresh;  // [max(n_pages, max_seqs)] free pages
    int32_t* mark;   // [max_seqs] list index of a slot
    int32_t* at;     // [max_seqs + 1] first fresh page of a list entry
    int32_t* keep;   // [max_seqs] a list entry's length
    int32_t* stage;  // [max_seqs][max_pages] new tables
};

__host__ __device__ inline int64_t book_words(int n_pages, int max_seqs, int max_pages) {
    const int64_t most = n_pages > max_seqs ? n_pages : max_seqs;
    return 16 + 3 * most + n_pages + 3 * (int64_t)max_seqs + 1 + (int64_t)max_seqs * max_pages;
}
__device__ __forceinline__ Book book_of(int32_t* p, const KvView& c) {
    const int64_t most = max(c.n_pages, c.max_seqs);
    Book b;
    b.head = p;
    b.from = p + 16;
    b.to = b.from + most;
    b.fresh = b.to + most;
    b.remap = b.fresh + most;
    b.mark = b.remap + c.n_pages;
    b.at = b.mark + c.max_seqs;
    b.keep = b.at + c.max_seqs + 1;
    b.stage = b.keep + c.max_seqs;
    return b;
}

constexpr int PLAN = 1024;  // threads of the one workgroup that does the bookkeeping

// Sum over the workgroup of every thread's v before it; total: of all.  Ends with a barrier.
__device__ __forceinline__ int scan(int v, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < PLAN / 64; ++w) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    __syncthreads();
    return before + x - v;
}

__device__ __forceinline__ int any(int v, int* lds) {  // workgroup-wide or
    int total;
    scan(v ? 1 : 0, lds, total);
    return total;
}

// One workgroup: global memory written before a barrier is read after it through the L2
__device__ __forceinline__ int peek(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void poke(int32_t* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// (its stores and atomics have reached the L2 once they are counted as done; peek reads there)
__device__ __forceinline__ void settle() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ int pages_of(const KvView& c, int64_t tokens) { return (int)((tokens + c.page_tokens - 1) / c.page_tokens); }
__device__ __forceinline__ bool slot_ok(const KvView& c, int s) { return s >= 0 && s < c.max_seqs; }
__device__ __forceinline__ bool len_ok(const KvView& c, int len) {
    return len >= 0 && (int64_t)len <= (int64_t)c.max_pages * c.page_tokens;
}

// Whether the list holds distinct slots with lengths in their limits
__device__ bool list_ok(const KvView& c, const Book& b, const int32_t* slots, int n, int* lds) {
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += PLAN) {
        const int s = slots[i];
        if (!slot_ok(c, s) || !len_ok(c, c.len[s]))
            bad = 1;
        else
            poke(&b.mark[s], n);
    }
    settle();
    for (int i = threadIdx.x; i < n; i += PLAN)
        if (slot_ok(c, slots[i])) atomicMin(&b.mark[slots[i]], i);
    settle();
    for (int i = threadIdx.x; i < n; i += PLAN)
        if (slot_ok(c, slots[i]) && peek(&b.mark[slots[i]]) != i) bad = 1;
    return !any(bad, lds);
}

// at[i] = sum of need(0) .. need(i - 1); returns the sum of all
template <typename F>
__device__ int place(const Book& b, int n, int* lds, F need) {
    int sum = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + threadIdx.x;
        int total;
        const int before = scan(i < n ? need(i) : 0, lds, total);
        if (i < n) b.at[i] = sum + before;
        sum += total;
    }
    return sum;
}

// The lowest `count` free pages into b.fresh; false if there are fewer
__device__ bool find_free(const KvView& c, const int32_t* ref, const Book& b, int64_t count, int* lds) {
    int64_t found = 0;
    for (int p0 = 0; p0 < c.n_pages && found < count; p0 += PLAN) {
        const int p = p0 + threadIdx.x;
        int total;
        const bool is_free = p < c.n_pages && peek(&ref[p]) == 0;
        const int before = scan(is_free ? 1 : 0, lds, total);
        if (is_free && found + before < count) b.fresh[found + before] = p;
        found += total;
    }
    settle();
    return found >= count;
}

__device__ __forceinline__ bool page_ok(const KvView& c, int p) { return p >= 0 && p < c.n_pages; }

struct PageArgs {
    KvView c;
    int32_t *ref, *scratch;
    const int32_t *a, *b;  // the operation's lists
    int n, layers;
    int64_t layer_codes, layer_scales;  // bytes of codes, words of scales in a layer
};

__device__ __forceinline__ void refuse(const KvView& c, const Book& b, int bit) {
    if (threadIdx.x == 0) {
        atomicOr(c.status, bit);
        b.head[0] = 0;
        b.head[1] = -1;
    }
}

__global__ __launch_bounds__(PLAN) void k_reserve(const PageArgs a) {
    __shared__ int lds[PLAN / 64];
    const KvView& c = a.c;
    const Book b = book_of(a.scratch, c);
    if (*c.status) return;
    if (!list_ok(c, b, a.a, a.n, lds)) return refuse(c, b, JX_KV_BAD_ARG);
    int bad = 0;
    for (int i = threadIdx.x; i < a.n; i += PLAN) {
        const int64_t add = a.b ? a.b[i] : 1;
        if (add < 0 || c.len[a.a[i]] + add > (int64_t)c.max_pages * c.page_tokens) bad = 1;
    }
    if (any(bad, lds)) return refuse(c, b, JX_KV_BAD_ARG);
    // (sums of needs stay below 2^31: n_pages_max * max_seqs is checked on the host)
    const int total = place(b, a.n, lds, [&](int i) {
        const int64_t len = c.len[a.a[i]];
        return pages_of(c, len + (a.b ? a.b[i] : 1)) - pages_of(c, len);
    });
    if (total && !find_free(c, a.ref, b, total, lds)) return refuse(c, b, JX_KV_NO_PAGES);
    settle();
    for (int i = threadIdx.x >> 6; i < a.n; i += PLAN / 64) {  // a wave per sequence
        const int slot = a.a[i], len = c.len[slot], add = a.b ? a.b[i] : 1;
        const int held = pages_of(c, len), need = pages_of(c, (int64_t)len + add) - held, at = peek(&b.at[i]);
        for (int k = threadIdx.x & 63; k < need; k += 64) {
            const int p = peek(&b.fresh[at + k]);
            c.table[(int64_t)slot * c.max_pages + held + k] = p;
            a.ref[p] = 1;
        }
        if ((threadIdx.x & 63) == 0) c.len[slot] = len + add;
    }
}

__global__ __launch_bounds__(PLAN) void k_trim(const PageArgs a) {
    __shared__ int lds[PLAN / 64];
    const KvView& c = a.c;
    const Book b = book_of(a.scratch, c);
    if (threadIdx.x == 0) b.head[0] = 0, b.head[1] = -1;
    if (*c.status) return;
    if (!list_ok(c, b, a.a, a.n, lds)) return refuse(c, b, JX_KV_BAD_ARG);
    auto target = [&](int i) { return a.b ? min(max(a.b[i], 0), c.len[a.a[i]]) : 0; };
    int bad = 0;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = wave; i < a.n; i += PLAN / 64)
        for (int k = max(0, pages_of(c, target(i)) - 1) + lane; k < pages_of(c, c.len[a.a[i]]); k += 64)
            if (!page_ok(c, c.table[(int64_t)a.a[i] * c.max_pages + k])) bad = 1;
    if (any(bad, lds)) return refuse(c, b, JX_KV_BAD_PAGE);
    auto drop = [&](int by) {
        for (int i = wave; i < a.n; i += PLAN / 64)
            for (int k = pages_of(c, target(i)) + lane; k < pages_of(c, c.len[a.a[i]]); k += 64)
                atomicAdd(&a.ref[c.table[(int64_t)a.a[i] * c.max_pages + k]], by);
    };
    drop(-1);
    settle();
    // a last page that is partly used and still shared becomes the sequence's own
    auto tail = [&](int i) -> int32_t* {
        const int len = target(i);
        return len % c.page_tokens ? &c.table[(int64_t)a.a[i] * c.max_pages + len / c.page_tokens] : nullptr;
    };
    const int total = place(b, a.n, lds, [&](int i) {
        const int32_t* t = tail(i);
        return t && peek(&a.ref[*t]) > 1 ? 1 : 0;
    });
    if (total && !find_free(c, a.ref, b, total, lds)) {
        drop(1);
        return refuse(c, b, JX_KV_NO_PAGES);
    }
    settle();
    for (int i = threadIdx.x; i < a.n; i += PLAN) {
        const int at = peek(&b.at[i]), next = i + 1 < a.n ? peek(&b.at[i + 1]) : total;
        const int len = target(i);
        if (next > at) {
            int32_t* t = tail(i);
            const int old = *t, p = peek(&b.fresh[at]);
            b.from[at] = old;
            b.to[at] = p;
            *t = p;
            atomicSub(&a.ref[old], 1);
            a.ref[p] = 1;
        }
        c.len[a.a[i]] = len;
    }
    if (threadIdx.x == 0) b.head[0] = total;
}

__global__ __launch_bounds__(PLAN) void k_fork(const PageArgs a) {
    __shared__ int lds[PLAN / 64];
    const KvView& c = a.c;
    const Book b = book_of(a.scratch, c);
    if (threadIdx.x == 0) b.head[0] = 0, b.head[1] = -1;
    if (*c.status) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int32_t *src = a.a, *dst = a.b;
    if (!list_ok(c, b, dst, a.n, lds)) return refuse(c, b, JX_KV_BAD_ARG);
    int bad = 0;
    for (int i = threadIdx.x; i < a.n; i += PLAN)
        if (!slot_ok(c, src[i]) || !len_ok(c, c.len[src[i]])) bad = 1;
    if (any(bad, lds)) return refuse(c, b, JX_KV_BAD_ARG);
    auto moves = [&](int i) { return src[i] != dst[i]; };
    // the new tables beside the old ones: a source may be a destination as well
    for (int i = wave; i < a.n; i += PLAN / 64) {
        const int len = c.len[src[i]];
        for (int k = lane; k < pages_of(c, len); k += 64) {
            const int p = c.table[(int64_t)src[i] * c.max_pages + k];
            b.stage[(int64_t)i * c.max_pages + k] = p;
            if (!page_ok(c, p)) bad = 1;
        }
        for (int k = lane; k < pages_of(c, c.len[dst[i]]); k += 64)
            if (!page_ok(c, c.table[(int64_t)dst[i] * c.max_pages + k])) bad = 1;
        if (lane == 0) b.keep[i] = len;
    }
    if (any(bad, lds)) return refuse(c, b, JX_KV_BAD_PAGE);
    const int total = place(b, a.n, lds, [&](int i) { return moves(i) && c.len[src[i]] % c.page_tokens ? 1 : 0; });
    if (total && !find_free(c, a.ref, b, total, lds)) return refuse(c, b, JX_KV_NO_PAGES);
    settle();
    for (int i = wave; i < a.n; i += PLAN / 64) {
        if (!moves(i)) continue;
        const int full = peek(&b.keep[i]) / c.page_tokens;
        for (int k = lane; k < full; k += 64) atomicAdd(&a.ref[peek(&b.stage[(int64_t)i * c.max_pages + k])], 1);
        for (int k = lane; k < pages_of(c, c.len[dst[i]]); k += 64) atomicSub(&a.ref[c.table[(int64_t)dst[i] * c.max_pages + k]], 1);
    }
    settle();
    for (int i = wave; i < a.n; i += PLAN / 64) {
        if (!moves(i)) continue;
        const int len = peek(&b.keep[i]), full = len / c.page_tokens;
        int32_t* row = c.table + (int64_t)dst[i] * c.max_pages;
        for (int k = lane; k < full; k += 64) row[k] = peek(&b.stage[(int64_t)i * c.max_pages + k]);
        if (lane == 0) {
            if (len % c.page_tokens) {
                const int at = peek(&b.at[i]), p = peek(&b.fresh[at]);
                b.from[at] = peek(&b.stage[(int64_t)i * c.max_pages + full]);
                b.to[at] = p;
                row[full] = p;
                a.ref[p] = 1;
            }
            c.len[dst[i]] = len;
        }
    }
    if (threadIdx.x == 0) b.head[0] = total;
}

__global__ __launch_bounds__(PLAN) void k_compact(const PageArgs a) {
    __shared__ int lds[PLAN / 64];
    const KvView& c = a.c;
    const Book b = book_of(a.scratch, c);
    if (threadIdx.x == 0) b.head[0] = 0, b.head[1] = -1;
    if (*c.status) return;
    int live = 0;
    for (int p = threadIdx.x; p < c.n_pages; p += PLAN) live += a.ref[p] > 0;
    int count;
    scan(live, lds, count);
    int high = 0, low = 0;
    for (int p0 = 0; p0 < c.n_pages; p0 += PLAN) {
        const int p = p0 + threadIdx.x;
        const bool held = p < c.n_pages && a.ref[p] > 0;
        const int is_high = held && p >= count, is_low = p < count && !held;
        int nh, nl;
        const int h = scan(is_high, lds, nh), l = scan(is_low, lds, nl);
        if (is_high) b.from[high + h] = p;
        if (is_low) b.to[low + l] = p;
        high += nh;
        low += nl;
    }
    settle();
    for (int i = threadIdx.x; i < high; i += PLAN) {  // as many free places below `count` as pages behind it
        const int from = peek(&b.from[i]), to = peek(&b.to[i]);
        b.remap[from] = to;
        a.ref[to] = a.ref[from];
        a.ref[from] = 0;
    }
    if (threadIdx.x == 0) {
        b.head[0] = high;
        b.head[1] = count;
        c.status[1] = count;
    }
}

// The copies that the bookkeeping listed, in every layer, and a compaction's new page numbers in the tables.  16 KB per workgroup
// and turn, all of it in flight: bound by HBM (957 MB read and written in 176 us, 5.4 TB/s, where a plain copy of 1 GiB
// reaches 5.24; 185 us without the non-temporal hints).
__global__ __launch_bounds__(256) void k_copy(const PageArgs a) {
    const KvView& c = a.c;
    const Book b = book_of(a.scratch, c);
    const int copies = b.head[0], count = b.head[1];
    const int64_t page_codes = 2LL * c.H * c.page_tokens * c.D;     // bytes, a multiple of 2048
    const int page_scales = 2 * c.H << c.blocks_shift;
    constexpr int SEG = 16384;
    const int segs = (int)((page_codes + SEG - 1) / SEG);
    const int64_t items = (int64_t)copies * a.layers * segs;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int seg = (int)(it % segs);
        const int layer = (int)(it / segs % a.layers), i = (int)(it / segs / a.layers);
        const int from = b.from[i], to = b.to[i];
        const int64_t at = (int64_t)seg * SEG, n = min((int64_t)SEG, page_codes - at);
        const uint8_t* s = reinterpret_cast<const uint8_t*>(c.codes) + layer * a.layer_codes + from * page_codes + at;
        uint8_t* d = reinterpret_cast<uint8_t*>(c.codes) + layer * a.layer_codes + to * page_codes + at;
        uint4 v[SEG / 4096];
#pragma unroll
        for (int k = 0; k < SEG / 4096; ++k)
            if (k * 4096 + threadIdx.x * 16 < n) v[k] = ld_stream16(s + k * 4096 + threadIdx.x * 16);
#pragma unroll
        for (int k = 0; k < SEG / 4096; ++k)
            if (k * 4096 + threadIdx.x * 16 < n) __builtin_nontemporal_store(u32x4{v[k].x, v[k].y, v[k].z, v[k].w}, reinterpret_cast<u32x4*>(d + k * 4096 + threadIdx.x * 16));
        if (seg == 0) {
            float* sc = c.scales + layer * a.layer_scales;
            for (int k = threadIdx.x; k < page_scales; k += 256) sc[(int64_t)to * page_scales + k] = sc[(int64_t)from * page_scales + k];
        }
    }
    if (copies > 0 && count >= 0) {
        const int64_t entries = (int64_t)c.max_seqs * c.max_pages;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
            const int slot = (int)(i / c.max_pages), k = (int)(i % c.max_pages);
            const int len = c.len[slot];
            if (!len_ok(c, len) || k >= pages_of(c, len)) continue;
            const int p = c.table[i];
            if (p >= count && p < c.n_pages) c.table[i] = b.remap[p];
        }
    }
}

// ---------------------------------------------------------------- checks of the host

#define REFUSE(cond, code, text) \
    do {                         \
        if (cond) return api_fail(code, text); \
    } while (0)

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_shape(const jx_kv_cache* c) {
    REFUSE(!c, JX_ERR_INVALID, "null cache");
    REFUSE(c->n_layers < 1 || c->n_pages < 1 || c->n_kv_heads < 1 || c->max_seqs < 1 || c->max_pages < 1, JX_ERR_INVALID,
           "a cache has at least one layer, page, kv head, slot and page of a slot");
    REFUSE(c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128 && c->page_tokens != 256, JX_ERR_UNSUPPORTED,
           "page_tokens is 32, 64, 128 or 256");
    REFUSE(c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32, JX_ERR_UNSUPPORTED,
           "head_dim is a multiple of 32 from 32 to 256");
    REFUSE(c->n_kv_heads > 65535, JX_ERR_UNSUPPORTED, "more than 65535 kv heads");
    REFUSE((int64_t)c->n_pages * 2 * c->n_kv_heads * (c->page_tokens / KV_BLOCK) > INT32_MAX, JX_ERR_UNSUPPORTED,
           "a layer has 2^31 blocks at most");
    REFUSE((int64_t)c->max_pages * c->page_tokens > KV_MAX_TOKENS, JX_ERR_UNSUPPORTED, "a sequence has 2^30 tokens at most");
    REFUSE((int64_t)c->max_seqs * c->max_pages > INT32_MAX, JX_ERR_UNSUPPORTED, "the table has 2^31 entries at most");
    return JX_OK;
}

int check_cache(const jx_kv_cache* c) {
    const int r = check_shape(c);
    if (r != JX_OK) return r;
    REFUSE(!c->codes || !c->scales || !c->table || !c->len || !c->ref || !c->status || !c->scratch, JX_ERR_INVALID,
           "null memory of the cache");
    REFUSE(!aligned(c->codes, 16), JX_ERR_INVALID, "codes are not 16-byte aligned");
    REFUSE(!aligned(c->scales, 4) || !aligned(c->table, 4) || !aligned(c->len, 4) || !aligned(c->ref, 4) || !aligned(c->status, 4) ||
               !aligned(c->scratch, 4), JX_ERR_INVALID, "memory of the cache is not aligned");
    return JX_OK;
}

int check_batch(const jx_kv_cache* c, const jx_kv_batch* b) {
    REFUSE(!b, JX_ERR_INVALID, "null batch");
    REFUSE(b->n_seqs < 0 || b->n_rows < 0 || b->max_rows < 0 || b->max_len < 0, JX_ERR_INVALID, "negative size of the batch");
    REFUSE(b->max_rows > b->n_rows, JX_ERR_INVALID, "max_rows is more than n_rows");
    REFUSE(!b->row_start && (b->n_rows != b->n_seqs || (b->n_seqs && b->max_rows < 1)), JX_ERR_INVALID,
           "without row_start every sequence has one row");
    REFUSE(!b->seqs && b->n_seqs > c->max_seqs, JX_ERR_INVALID, "more sequences than slots");
    REFUSE(b->max_rows > KV_MAX_TOKENS, JX_ERR_UNSUPPORTED, "a sequence has 2^30 rows at most");
    REFUSE(!aligned(b->seqs, 4) || !aligned(b->row_start, 4), JX_ERR_INVALID, "a list is not aligned");
    return JX_OK;
}

size_t type_size(int t) { return t == JX_TYPE_F32 ? 4 : t == JX_TYPE_F16 || t == JX_TYPE_BF16 ? 2 : 0; }

KvView view(const jx_kv_cache* c, int layer) {
    KvView v;
    const int shift = __builtin_ctz((unsigned)c->page_tokens) - 5;
    const int64_t blocks = ((int64_t)c->n_pages * 2 * c->n_kv_heads) << shift;
    v.codes = c->codes + (int64_t)layer * blocks * KV_BLOCK * c->head_dim;
    v.scales = c->scales + (int64_t)layer * blocks;
    v.table = c->table;
    v.len = c->len;
    v.status = c->status;
    v.n_pages = c->n_pages;
    v.page_tokens = c->page_tokens;
    v.blocks_shift = shift;
    v.H = c->n_kv_heads;
    v.D = c->head_dim;
    v.max_seqs = c->max_seqs;
    v.max_pages = c->max_pages;
    return v;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? JX_OK : api_fail(JX_ERR_HIP, std::string("launch: ") + hipGetErrorString(e));
}

template <typename K>
int page_operation(K kernel, bool copies, const jx_kv_cache* c, const int32_t* x, const int32_t* y, int n, void* stream) {
    const int r = api_device(c->device);
    if (r != JX_OK) return r;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    PageArgs a;
    a.c = view(c, 0);
    a.ref = c->ref;
    a.scratch = c->scratch;
    a.a = x;
    a.b = y;
    a.n = n;
    a.layers = c->n_layers;
    a.layer_scales = ((int64_t)c->n_pages * 2 * c->n_kv_heads) << a.c.blocks_shift;
    a.layer_codes = a.layer_scales * KV_BLOCK * c->head_dim;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(PLAN), 0, st, a);
    if (copies) hipLaunchKernelGGL(k_copy, dim3(2048), dim3(256), 0, st, a);
    return launched();
}

int check_list(const jx_kv_cache* c, const int32_t* slots, int n) {
    const int r = check_cache(c);
    if (r != JX_OK) return r;
    REFUSE(n < 0, JX_ERR_INVALID, "negative count");
    REFUSE(n > c->max_seqs, JX_ERR_INVALID, "more entries than slots");
    REFUSE(n && !slots, JX_ERR_INVALID, "null list");
    REFUSE(!aligned(slots, 4), JX_ERR_INVALID, "a list is not aligned");
    return JX_OK;
}

int check_attention(const jx_kv_cache* c, const jx_kv_batch* b, const jx_attention* t) {
    int r = check_shape(c);
    if (r == JX_OK) r = check_batch(c, b);
    if (r != JX_OK) return r;
    REFUSE(!t, JX_ERR_INVALID, "null attention");
    REFUSE(!type_size(t->type), JX_ERR_UNSUPPORTED, "q and out are F32, F16 or BF16");
    REFUSE(t->n_heads < 1 || t->n_heads % c->n_kv_heads, JX_ERR_INVALID, "n_heads is a multiple of the cache's kv heads");
    REFUSE((int64_t)b->max_rows * (t->n_heads / c->n_kv_heads) > KV_MAX_TOKENS, JX_ERR_UNSUPPORTED,
           "a sequence has 2^30 rows times heads of a group at most");
    REFUSE(!(t->scale - t->scale == 0.0f), JX_ERR_INVALID, "scale is not finite");
    REFUSE(!(t->softcap >= 0.0f) || !(t->softcap - t->softcap == 0.0f), JX_ERR_INVALID, "softcap is negative or not finite");
    REFUSE(t->window < 0, JX_ERR_INVALID, "negative window");
    REFUSE(t->causal != 0 && t->causal != 1, JX_ERR_INVALID, "causal is 0 or 1");
    REFUSE(!aligned(t->alibi, 4), JX_ERR_INVALID, "alibi is not aligned");
    const int64_t width = (int64_t)t->n_heads * c->head_dim;
    REFUSE((t->q_stride && t->q_stride < width) || (t->out_stride && t->out_stride < width), JX_ERR_INVALID,
           "a row stride is smaller than a row");
    return JX_OK;
}

size_t workspace(const jx_kv_cache* c, const AttendPlan& p) {
    return (size_t)p.partials * p.rows_cap * (c->head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace jx

using namespace jx;

extern "C" {

int64_t jx_kv_scratch_words(const jx_kv_cache* c) {
    return check_shape(c) == JX_OK ? book_words(c->n_pages, c->max_seqs, c->max_pages) : 0;
}

int jx_kv_reserve(const jx_kv_cache* c, const int32_t* slots, const int32_t* n_new, int32_t n, void* stream) {
    const int r = check_list(c, slots, n);
    if (r != JX_OK || n == 0) return r;
    REFUSE(!aligned(n_new, 4), JX_ERR_INVALID, "a list is not aligned");
    return page_operation(k_reserve, false, c, slots, n_new, n, stream);
}

int jx_kv_trim(const jx_kv_cache* c, const int32_t* slots, const int32_t* new_len, int32_t n, void* stream) {
    const int r = check_list(c, slots, n);
    if (r != JX_OK || n == 0) return r;
    REFUSE(!aligned(new_len, 4), JX_ERR_INVALID, "a list is not aligned");
    return page_operation(k_trim, new_len != nullptr, c, slots, new_len, n, stream);
}

int jx_kv_fork(const jx_kv_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    int r = check_list(c, src, n);
    if (r == JX_OK) r = check_list(c, dst, n);
    if (r != JX_OK || n == 0) return r;
    return page_operation(k_fork, true, c, src, dst, n, stream);
}

int jx_kv_compact(const jx_kv_cache* c, void* stream) {
    const int r = check_cache(c);
    if (r != JX_OK) return r;
    return page_operation(k_compact, true, c, nullptr, nullptr, 0, stream);
}

int jx_kv_append(const jx_kv_cache* c, const jx_kv_batch* b, int32_t layer, int32_t type, const void* k, const void* v,
                 int64_t row_stride, void* stream) {
    int r = check_cache(c);
    if (r == JX_OK) r = check_batch(c, b);
    if (r != JX_OK) return r;
    REFUSE(layer < 0 || layer >= c->n_layers, JX_ERR_INVALID, "no such layer");
    const size_t size = type_size(type);
    REFUSE(!size, JX_ERR_UNSUPPORTED, "k and v are F32, F16 or BF16");
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
    REFUSE(row_stride && row_stride < width, JX_ERR_INVALID, "the row stride is smaller than a row");
    if (b->n_seqs == 0 || b->max_rows == 0) return JX_OK;
    REFUSE(!k || !v, JX_ERR_INVALID, "null k or v");
    REFUSE(!aligned(k, size) || !aligned(v, size), JX_ERR_INVALID, "k or v is not aligned");
    AppendArgs a;
    a.blocks = (b->max_rows + KV_BLOCK - 2) / KV_BLOCK + 1;
    REFUSE((int64_t)b->n_seqs * a.blocks > INT32_MAX, JX_ERR_UNSUPPORTED, "the batch is too large for one call");
    r = api_device(c->device);
    if (r != JX_OK) return r;
    a.c = view(c, layer);
    a.b = KvRows{b->seqs, b->row_start, b->n_seqs, b->n_rows, b->max_rows};
    a.ref = c->ref;
    a.k = k;
    a.v = v;
    a.stride = row_stride ? row_stride : width;
    a.vec = aligned(k, 16) && aligned(v, 16) && a.stride * size % 16 == 0;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (type == JX_TYPE_F32)
        append_type<float>(a, st);
    else if (type == JX_TYPE_F16)
        append_type<_Float16>(a, st);
    else
        append_type<__bf16>(a, st);
    return launched();
}

size_t jx_kv_attention_workspace(const jx_kv_cache* c, const jx_kv_batch* b, const jx_attention* t) {
    if (check_attention(c, b, t) != JX_OK || b->n_seqs == 0 || b->max_rows == 0) return 0;
    return workspace(c, attend_plan(*c, *b, *t));
}

int jx_kv_attention(const jx_kv_cache* c, const jx_kv_batch* b, const jx_attention* t, int32_t layer, const void* q, void* out,
                    void* ws, size_t ws_bytes, void* stream) {
    int r = check_cache(c);
    if (r == JX_OK) r = check_attention(c, b, t);
    if (r != JX_OK) return r;
    REFUSE(layer < 0 || layer >= c->n_layers, JX_ERR_INVALID, "no such layer");
    if (b->n_seqs == 0 || b->max_rows == 0) return JX_OK;
    REFUSE(!q || !out, JX_ERR_INVALID, "null q or out");
    const size_t size = type_size(t->type);
    REFUSE(!aligned(q, size) || !aligned(out, size), JX_ERR_INVALID, "q or out is not aligned");
    const AttendPlan p = attend_plan(*c, *b, *t);
    const size_t need = workspace(c, p);
    REFUSE(need && (!ws || ws_bytes < need), JX_ERR_INVALID, "the workspace is smaller than jx_kv_attention_workspace()");
    REFUSE(need && !aligned(ws, 16), JX_ERR_INVALID, "the workspace is not 16-byte aligned");
    REFUSE((int64_t)b->n_seqs * p.splits * p.row_tiles * c->n_kv_heads > INT32_MAX, JX_ERR_UNSUPPORTED,
           "the batch is too large for one call");
    r = api_device(c->device);
    if (r != JX_OK) return r;
    AttendArgs a;
    a.c = view(c, layer);
    a.b = KvRows{b->seqs, b->row_start, b->n_seqs, b->n_rows, b->max_rows};
    a.q = q;
    a.out = out;
    const int64_t width = (int64_t)t->n_heads * c->head_dim;
    a.q_stride = t->q_stride ? t->q_stride : width;
    a.out_stride = t->out_stride ? t->out_stride : width;
    a.alibi = t->alibi;
    a.part_o = static_cast<float*>(ws);
    a.part_ml = a.part_o + (size_t)p.partials * p.rows_cap * c->head_dim;
    a.type = t->type;
    a.heads = t->n_heads;
    a.G = t->n_heads / c->n_kv_heads;
    a.scale = std::fabs(t->scale);
    a.scale2 = a.scale * 1.44269504088896340736f;
    a.flip = std::signbit(t->scale);
    a.cap = t->softcap;
    a.window = std::min(t->window, KV_MAX_TOKENS);
    a.causal = t->causal;
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.waves = p.waves;
    a.group = p.group;
    a.tile_rows = p.tile_rows;
    a.row_tiles = p.row_tiles;
    a.rows_cap = p.rows_cap;
    a.q_vec = aligned(q, 16) && a.q_stride * size % 16 == 0;
    a.out_vec = aligned(out, 16) && a.out_stride * size % 16 == 0;
    launch_attend(a, reinterpret_cast<hipStream_t>(stream));
    return launched();
}

}  // extern "C"
