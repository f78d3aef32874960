// A step over a paged KV cache, as the kernels see it: new rows of many sequences, one sequence's rows behind another's,
// and pages of a power of two tokens.  All of it lies on the device, so that a recorded launch serves any step.
//
// Nothing here trusts what the arrays hold with memory: offsets are clamped to the rows, lengths to the page table's width,
// pages to the cache.  Offsets that decrease would have more blocks than attention's launch has workgroups: it finds them and
// takes every row for nobody's.  (The append takes a row for the first sequence's whose offsets enclose it.)
#pragma once

#include "l3_device.hpp"
#include "l3_host.hpp"

namespace l3 {

struct PagedStep {
    const int* q_offsets;   // rows of sequence b: q_offsets[b] .. q_offsets[b + 1]
    const int* kv_lens;     // tokens of sequence b in the cache, those of its new rows included
    const int* table;       // page of tokens i * page size ... of sequence b: table[b * table_stride + i]
    int64_t table_stride;
    int rows, seqs, pages, page_shift;
    int max_kv;             // tokens that a row of the table covers
};

// A row's sequence (-1: it belongs to none, or its position is negative) and its position there.
struct RowPlace {
    int seq, pos;
};

// The place of a row, for a wavefront; the same in every lane.  A lane looks at four sequences at once, so that up to 256 of
// them cost one trip to memory.
__device__ __forceinline__ RowPlace place_of_row(const PagedStep& s, int row) {
    const int lane = threadIdx.x & (kWaveSize - 1);
    for (int base = 0; base < s.seqs; base += 4 * kWaveSize) {
        int from[4], to[4], len[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = min(base + i * kWaveSize + lane, s.seqs - 1);
            from[i] = s.q_offsets[b];
            to[i] = s.q_offsets[b + 1];
            len[i] = s.kv_lens[b];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t here = __builtin_amdgcn_ballot_w64(base + i * kWaveSize + lane < s.seqs && from[i] <= row && row < to[i]);
            if (here) {
                const int at = __builtin_ctzll(here);
                const int end = min(__builtin_amdgcn_readlane(to[i], at), s.rows);
                const int kv = min(__builtin_amdgcn_readlane(len[i], at), s.max_kv);
                const int pos = kv - end + row;
                return {pos >= 0 ? base + i * kWaveSize + at : -1, pos};
            }
        }
    }
    return {-1, -1};
}

// First element of token t of sequence b in a cache with {page, token} strides.  (t < max_kv)
__device__ __forceinline__ int64_t paged_token(const PagedStep& s, int b, int t, int64_t page_stride, int64_t token_stride) {
    const int page = s.table[int64_t(b) * s.table_stride + (t >> s.page_shift)];
    return int64_t(min(max(page, 0), s.pages - 1)) * page_stride + int64_t(t & ((1 << s.page_shift) - 1)) * token_stride;
}

struct PagedAttnParams {
    PagedStep step;
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t q_sr, q_sh, k_sp, k_st, k_sh, v_sp, v_st, v_sh, o_sr, o_sh;
    int QH, KVH;
    int R, positions;   // query heads to a kv head; positions that 16 columns hold
    int inverse;        // column / R is column * inverse >> 8 for columns below 16
    double per_position;   // 1 / positions
    int max_new;   // most rows of a sequence as the caller says, 0: it does not (chooses between forms, never what is computed)
    float scale_log2e;
};

bool attn_paged_fits(const PagedStep& step, int QH, int KVH, int HD, int max_new);   // in a launch
size_t attn_paged_workspace_bytes(const PagedStep& step, int QH, int KVH, int HD, int max_new);
int launch_attn_paged(const PagedAttnParams& p, int HD, void* workspace, hipStream_t stream);
int launch_rot_embed_append_paged(const PagedStep& step, const void* qkv, int64_t qkv_stride, const float* table, int table_rows,
                                  const void* q_weight, const void* k_weight, float eps, void* q_out, void* k_pages, void* v_pages,
                                  const int64_t* k_strides, const int64_t* v_strides, int NH, int KVH, int HD, hipStream_t stream);
int launch_norm_rot_embed(const void* q, const void* k, const void* q_weight, const void* k_weight, float eps, const float* freq,
                          void* q_out, void* k_out, int B, int T, int NH, int KVH, int HD, const int64_t* q_strides,
                          const int64_t* k_strides, hipStream_t stream);

}  // namespace l3
