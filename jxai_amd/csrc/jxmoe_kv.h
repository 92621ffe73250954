// The paged 8-bit key/value cache: what its kernels (kv.hip, attend.hip) and the C entry points share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/jxmoe.h"

namespace jx {

constexpr int KV_BLOCK = JX_KV_BLOCK;
constexpr int KV_MAX_TOKENS = 1 << 30;  // of one sequence: positions and windows add and subtract in 32 bits

// Error text and device of the calling thread (runtime.hip).
int api_fail(int code, const std::string& msg);
int api_device(int device);  // current, if jx_moe_init has been called for it

// The cache as a kernel sees it.  codes / scales begin at the layer of the call.
struct KvView {
    int8_t* codes;
    float* scales;
    int32_t *table, *len, *status;
    int n_pages, page_tokens, blocks_shift;  // page_tokens = 32 << blocks_shift
    int H, D, max_seqs, max_pages;
    // block number of (page, K or V, head, block of the page); its codes are 32 * D bytes at this times 32 * D
    __host__ __device__ int block_index(int page, int which, int head, int block) const {
        return (((page * 2 + which) * H + head) << blocks_shift) + block;
    }
};

struct KvRows {
    const int32_t *seqs, *row_start;
    int n_seqs, n_rows, max_rows;
};

struct KvSeq {
    int slot, len, row0, n;  // n = 0: nothing to do
};

// Sequence i of a batch with everything in its limits; otherwise no rows, and the status word says so.
__device__ __forceinline__ KvSeq kv_seq(const KvView& c, const KvRows& b, int i) {
    KvSeq s;
    s.slot = b.seqs ? b.seqs[i] : i;
    const int r0 = b.row_start ? b.row_start[i] : i;
    const int r1 = b.row_start ? b.row_start[i + 1] : i + 1;
    const bool slot_ok = s.slot >= 0 && s.slot < c.max_seqs;
    s.len = slot_ok ? c.len[s.slot] : 0;
    const bool ok = slot_ok && r0 >= 0 && r0 <= r1 && r1 <= b.n_rows && r1 - r0 <= b.max_rows && s.len >= 0 &&
                    (int64_t)s.len <= (int64_t)c.max_pages * c.page_tokens;
    s.row0 = r0;
    s.n = ok ? r1 - r0 : 0;
    if (!ok) atomicOr(c.status, JX_KV_BAD_ARG);
    return s;
}

struct AttendArgs {
    KvView c;
    KvRows b;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const float* alibi;
    float* part_o;   // [partials][rows_cap][D] sums of weights times values
    float* part_ml;  // [partials][rows_cap][2] the running maximum and the sum of weights
    int type, heads, G;
    float scale;     // |softmax scale|
    float scale2;    // |softmax scale| * log2(e)
    bool flip;       // it is negative
    float cap;       // 0: none (natural units)
    int window, causal;
    int chunk;       // tiles of 32 tokens that a workgroup takes at most, unless that makes more than `splits` of a sequence
    int splits;
    int waves;       // k_attend_stream: waves of the launch
    int group;       //   waves whose parts become one partial
    int tile_rows;   // rows of a row tile; more than 32: k_attend_rows
    int row_tiles;   // of the sequence with the most rows
    int rows_cap;    // rows of a row tile at most: min(tile_rows, max_rows * G)
    bool q_vec, out_vec;  // 16-byte aligned rows
};

// How many splits the launch for this batch takes, and its chunk; the workspace is sized by it.
struct AttendPlan {
    int splits, chunk, tile_rows, row_tiles, rows_cap;
    int waves, group;  // waves not 0: k_attend_stream
    int64_t partials;  // of the workspace, each rows_cap rows of D + 2 floats
};
AttendPlan attend_plan(const jx_kv_cache& c, const jx_kv_batch& b, const jx_attention& a);
void launch_attend(const AttendArgs& a, hipStream_t st);

}  // namespace jx
