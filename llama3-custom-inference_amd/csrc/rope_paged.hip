// Rotary embedding of query and key heads with a norm of every head in front, and the rotary embedding of a step's ragged
// rows with the rotated keys and the values written into a paged cache.  Extensions of custom_kernels.cu:391-442 and
// model.py:100-106.
//
//   n(x) = x / sqrt(mean(x^2) + eps) * w    (a head's HD values; only where there are norm weights)
//   y[2i] = n[2i] cos - n[2i+1] sin,  y[2i+1] = n[2i] sin + n[2i+1] cos
//
// float32 throughout and one rounding.  The rotation is linear, so the norm's factor goes behind it: x w is exact in float32
// (two bf16 factors), its rotation is off by a few 2^-24 of the result also where the two products cancel, and so is the
// scaled result; a norm rounded to float32 in front would leave 2^-24 of the larger product in a small difference.
// A lane holds a 16-byte chunk of a head (four pairs), the HD / 8 lanes of a head lie side by side, and the sum of squares
// goes through DPP within them.
#include "paged.hpp"

namespace l3 {

namespace {

constexpr int kThreads = 256;

// Rotation of a chunk, behind the norm of its head where `w` says so.  (All lanes of a head come here together.)
template <int VPR>
__device__ __forceinline__ uint4 norm_rotate(const uint4& xv, bool normed, const uint4& wv, float eps, const float4& f0, const float4& f1) {
    if (!normed) {
        return make_uint4(rotate_pair(xv.x, f0.x, f0.y), rotate_pair(xv.y, f0.z, f0.w), rotate_pair(xv.z, f1.x, f1.y),
                          rotate_pair(xv.w, f1.z, f1.w));
    }
    float x[8], w[8], sum = 0.f;
    unpack8(xv, x);
    unpack8(wv, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    const float scale = 1.0f / sqrtf(group_sum<VPR>(sum) * (1.0f / (VPR * 8)) + eps);
    const float c[4] = {f0.x, f0.z, f1.x, f1.z}, s[4] = {f0.y, f0.w, f1.y, f1.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 y = rotate_floats(x[2 * i] * w[2 * i], x[2 * i + 1] * w[2 * i + 1], c[i], s[i]);
        o[i] = pack_bf16x2(y.x * scale, y.y * scale);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

struct AppendParams {
    PagedStep step;
    const uint16_t* qkv;
    const float* table;
    const uint16_t *q_weight, *k_weight;
    uint16_t *q_out, *k_pages, *v_pages;
    int64_t qkv_stride, k_sp, k_st, k_sh, v_sp, v_st, v_sh;
    int NH, KVH, table_rows;
    float eps;
};

// A workgroup has one row; a thread the same chunk of every (256 / VPR)th head.  Bound by bytes: four prompts of 1500 to 2600
// tokens, 32/8 heads of 128, 192 MB in 34 us (5.6 TB/s; the counters show 98 MB read and 94 written); pieces of 1 to 601
// tokens, 28 MB, 9 us, of which 3 are the launch and the way to the first load: place, page and row are three trips to memory, which
// other rows' workgroups cover (rows requested ahead of their place: no faster).  A single row: 2.2 us.
template <int HD>
__global__ void __launch_bounds__(kThreads) rot_embed_append_paged_kernel(const AppendParams p) {
    constexpr int VPR = HD / 8, HEADS = kThreads / VPR;
    const int row = blockIdx.x;
    const int c = threadIdx.x % VPR, h0 = threadIdx.x / VPR;
    const RowPlace place = place_of_row(p.step, row);
    const int slots = p.NH + 2 * p.KVH;
    const bool there = place.seq >= 0 && place.pos < p.table_rows;
    if (!there) {   // the row belongs to no token: its queries are zeros, and nothing is written to the cache
        for (int h = h0; h < p.NH; h += HEADS) store16(p.q_out + (int64_t(row) * p.NH + h) * HD + c * 8, make_uint4(0u, 0u, 0u, 0u));
        return;
    }
    const float4* fp = reinterpret_cast<const float4*>(p.table + int64_t(place.pos) * HD + c * 8);
    const float4 f0 = fp[0], f1 = fp[1];
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    const uint4 wq = p.q_weight ? load16(p.q_weight + c * 8) : none, wk = p.k_weight ? load16(p.k_weight + c * 8) : none;
    uint16_t* const k_row = p.k_pages + paged_token(p.step, place.seq, place.pos, p.k_sp, p.k_st) + c * 8;
    uint16_t* const v_row = p.v_pages + paged_token(p.step, place.seq, place.pos, p.v_sp, p.v_st) + c * 8;
    for (int h = h0; h < slots; h += HEADS) {
        const uint4 xv = load16_stream(p.qkv + row * p.qkv_stride + int64_t(h) * HD + c * 8);
        if (h < p.NH) {
            store16(p.q_out + (int64_t(row) * p.NH + h) * HD + c * 8, norm_rotate<VPR>(xv, p.q_weight != nullptr, wq, p.eps, f0, f1));
        } else if (h < p.NH + p.KVH) {
            store16(k_row + (h - p.NH) * p.k_sh, norm_rotate<VPR>(xv, p.k_weight != nullptr, wk, p.eps, f0, f1));
        } else {
            store16(v_row + (h - p.NH - p.KVH) * p.v_sh, xv);
        }
    }
}

struct NormRopeParams {
    const uint16_t *q, *k, *q_weight, *k_weight;
    const float* freq;
    uint16_t *q_out, *k_out;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
    int T, NH, KVH;
    float eps;
};

// A workgroup has one row of a sequence (blockIdx.x: token, y: sequence).  Bound by bytes: 2 x 2039 tokens, 32/8 heads of 128, 85 MB
// in 17.6 us (4.8 TB/s; four chunks of a thread in flight: 19.2).  64 sequences' single tokens: 3.4 us.
template <int HD>
__global__ void __launch_bounds__(kThreads) norm_rot_embed_kernel(const NormRopeParams p) {
    constexpr int VPR = HD / 8, HEADS = kThreads / VPR;
    const int t = blockIdx.x;
    const int64_t b = blockIdx.y;
    const int c = threadIdx.x % VPR, h0 = threadIdx.x / VPR;
    const float4* fp = reinterpret_cast<const float4*>(p.freq + int64_t(t) * HD + c * 8);
    const float4 f0 = fp[0], f1 = fp[1];
    const uint4 wq = load16(p.q_weight + c * 8), wk = load16(p.k_weight + c * 8);
    for (int h = h0; h < p.NH + p.KVH; h += HEADS) {
        if (h < p.NH) {
            const uint4 xv = load16_stream(p.q + b * p.q_sb + t * p.q_st + h * p.q_sh + c * 8);
            store16(p.q_out + ((b * p.T + t) * p.NH + h) * HD + c * 8, norm_rotate<VPR>(xv, true, wq, p.eps, f0, f1));
        } else {
            const int hk = h - p.NH;
            const uint4 xv = load16_stream(p.k + b * p.k_sb + t * p.k_st + hk * p.k_sh + c * 8);
            store16(p.k_out + ((b * p.T + t) * p.KVH + hk) * HD + c * 8, norm_rotate<VPR>(xv, true, wk, p.eps, f0, f1));
        }
    }
}

}  // namespace

int launch_rot_embed_append_paged(const PagedStep& step, const void* qkv, int64_t qkv_stride, const float* table, int table_rows,
                                  const void* q_weight, const void* k_weight, float eps, void* q_out, void* k_pages, void* v_pages,
                                  const int64_t* k_strides, const int64_t* v_strides, int NH, int KVH, int HD, hipStream_t stream) {
    AppendParams p;
    p.step = step;
    p.qkv = static_cast<const uint16_t*>(qkv);
    p.table = table;
    p.q_weight = static_cast<const uint16_t*>(q_weight);
    p.k_weight = static_cast<const uint16_t*>(k_weight);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.k_pages = static_cast<uint16_t*>(k_pages);
    p.v_pages = static_cast<uint16_t*>(v_pages);
    p.qkv_stride = qkv_stride;
    p.k_sp = k_strides[0]; p.k_st = k_strides[1]; p.k_sh = k_strides[2];
    p.v_sp = v_strides[0]; p.v_st = v_strides[1]; p.v_sh = v_strides[2];
    p.NH = NH; p.KVH = KVH; p.table_rows = table_rows; p.eps = eps;
    const dim3 grid(unsigned(step.rows)), block(kThreads);
    return HD == 64 ? enqueue(rot_embed_append_paged_kernel<64>, grid, block, 0, stream, p)
                    : enqueue(rot_embed_append_paged_kernel<128>, grid, block, 0, stream, p);
}

int launch_norm_rot_embed(const void* q, const void* k, const void* q_weight, const void* k_weight, float eps, const float* freq,
                          void* q_out, void* k_out, int B, int T, int NH, int KVH, int HD, const int64_t* q_strides,
                          const int64_t* k_strides, hipStream_t stream) {
    NormRopeParams p;
    p.q_weight = static_cast<const uint16_t*>(q_weight);
    p.k_weight = static_cast<const uint16_t*>(k_weight);
    p.freq = freq;
    p.q_sb = q_strides[0]; p.q_st = q_strides[1]; p.q_sh = q_strides[2];
    p.k_sb = k_strides[0]; p.k_st = k_strides[1]; p.k_sh = k_strides[2];
    p.T = T; p.NH = NH; p.KVH = KVH; p.eps = eps;
    for (int b0 = 0; b0 < B; b0 += 65535) {   // (a grid's second dimension)
        p.q = static_cast<const uint16_t*>(q) + b0 * p.q_sb;
        p.k = static_cast<const uint16_t*>(k) + b0 * p.k_sb;
        p.q_out = static_cast<uint16_t*>(q_out) + int64_t(b0) * T * NH * HD;
        p.k_out = static_cast<uint16_t*>(k_out) + int64_t(b0) * T * KVH * HD;
        const dim3 grid(unsigned(T), unsigned(B - b0 < 65535 ? B - b0 : 65535)), block(kThreads);
        const int rc = HD == 64 ? enqueue(norm_rot_embed_kernel<64>, grid, block, 0, stream, p)
                                : enqueue(norm_rot_embed_kernel<128>, grid, block, 0, stream, p);
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace l3
