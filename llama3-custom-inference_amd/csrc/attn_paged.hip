// Causal grouped-query attention of ragged rows over a paged KV cache.
//
//   out[row, h] = sum_{j <= p} softmax_j(scale q[row, h] . k_j) v_j,   p = position of the row in its sequence
//
// Columns of the matrix tiles are (position, query head) pairs of one kv head, as in the dense kernels: 16 / R consecutive
// positions of the R query heads in a block of 16.
//   S[tokens x 16 columns] = K Q^T,   O^T[dims x 16 columns] += V^T P     (v_mfma_f32_16x16x32_bf16)
//
// Softmax with a running maximum: scores, maxima, sums and outputs are float32; the weights exp(s - m) alone are rounded, to the
// bf16 that the matrix instructions take (2^-9 of a weight, errors of all tokens independent: below the rounding of the output;
// over N(0, 1) values 0.0020 to 0.0023 of the result's norm in all, 0.0016 to 0.0017 with float32 weights).  The denominator is a float32 sum,
// in the narrow form of the weights before that rounding, as in the dense decode kernels, in the wide form of the rounded ones,
// which the matrix pipe adds up on its way.
//
// A block is what one workgroup of four wavefronts takes.  Narrow: 16 or 32 columns, whose tokens the wavefronts share out
// among themselves, each with a softmax of its own (a sequence with a single or a few new tokens, bound by the bytes of its
// keys and values).  Wide: 64 or 128 columns, 16 or 32 to a wavefront, all against one stream of tokens in LDS (a prompt's
// piece, bound by the matrix pipe).  A call takes the one form or the other by the most rows that a sequence has: beside a
// prompt's piece the few columns of other sequences are wide blocks too, whose idle wavefronts load tokens all the same.
//
// Lengths differ from sequence to sequence by orders of magnitude and lie on the device, so the work is shared out there, by
// every workgroup for itself and alike:
//   narrow  every block weighs its tokens (and a constant), the weights of all blocks, kv head by kv head, form one line, and
//           part c of n takes the line from c / n to (c + 1) / n, cut at whole tiles;
//   wide    blocks are work items in order of their length; where a few of them would outlast all others, blocks longer
//           than a fair share are cut into pieces.
// A block that is cut leaves partial results (running maximum, sum, unnormalised output; float32), and a last launch adds them
// up.  No workgroup waits for another.
#include <algorithm>

#include "attn_common.hpp"
#include "attn_mfma_core.hpp"
#include "paged.hpp"

namespace l3 {

namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWaveSize;
constexpr int kTile = 64;                            // tokens between two places where a block may be cut
constexpr int kBlockWeight = 192;                    // what a narrow block costs beside its tokens, in tokens
constexpr int kLeastChunk = 256;                     // weight below which the line is not divided further
constexpr int kLeastPiece = 64;                      // tokens below which a piece goes to its neighbour
constexpr int kLeastCut = 512;                       // tokens that a page table has to hold for narrow blocks to be cut
constexpr int kLeastWideCut = 24 * kTile;            // ... for wide ones
constexpr float kNothing = kMaskedScore;             // a running maximum before any score
constexpr int kXcds = 8;
constexpr int kLeastWidePiece = 8;                   // tiles (a piece's start and its partial result cost some 5)
constexpr int kUncut = 1 << 28;                      // tiles: more than there are

// A partial result: as a wide block's registers lie, or a narrow block's columns one after the other.
constexpr int wide_slot_bytes(int HD, int CB) { return CB * (HD + 8) * 4 * kWaveSize; }
constexpr int narrow_slot_bytes(int HD, int CB) { return CB * 16 * (HD + 2) * 4 + 128 * CB; }

// A block that was cut, as the last launch finds it: written by the workgroup that has its first piece.
struct __align__(16) CutBlock {
    int pieces;              // 0: no block that was cut begins here; narrow: 1, the parts behind it say where it ends
    int row, rows, kvh;
    int first, next, stride; // slot of the first piece, and of the second: the others follow it in steps of `stride`
    int ends;                // narrow: the block that was begun by an earlier part ends in this one
};

// What a launch has beside the arguments.
struct PagedGrid {
    char* slots;      // partial results; null: nothing is cut
    CutBlock* cuts;   // entry 0: how many there are behind it (in `pieces`); one for each narrow part, or piece of a wide block
    int entries;      // of them, at most
    int units;        // compute units
};

// A sequence, as its blocks see it.
struct Sequence {
    int row, n, kv;   // first row, rows, tokens
    int blocks;
    bool falls;       // its offsets decrease
    __device__ __forceinline__ int past() const { return max(kv - n, 0); }
    // weight of the first j blocks
    __device__ __forceinline__ int64_t weight(int j, int positions) const {
        return int64_t(j) * (past() + kBlockWeight) + int64_t(positions) * (int64_t(j) * (j + 1) / 2);
    }
    // tokens that block j's last row sees
    __device__ __forceinline__ int tokens(int j, int positions) const { return max(kv - n + min(n, (j + 1) * positions), 0); }
};

// A step of a prefix operation over a wavefront: x combined with what lies 1, 2, 4, 8 lanes before within 16, and with the last
// of the 16 or 32 lanes before that; 0 where there is nothing.
template <typename F>
__device__ __forceinline__ void wave_prefix(F step) {
    using std::integral_constant;
    step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr:1, 2, 4, 8
    step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // row_bcast:15 into rows 1 and 3
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});   // row_bcast:31 into rows 2 and 3
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int before(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x) {
    wave_prefix([&](auto ctrl, auto rows) { x += before<decltype(ctrl)::value, decltype(rows)::value>(x); });
    return x;
}
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
    wave_prefix([&](auto ctrl, auto rows) {
        const uint32_t lo = before<decltype(ctrl)::value, decltype(rows)::value>(int(uint32_t(x)));
        const uint32_t hi = before<decltype(ctrl)::value, decltype(rows)::value>(int(uint32_t(uint64_t(x) >> 32)));
        x += int64_t(uint64_t(hi) << 32 | lo);
    });
    return x;
}
__device__ __forceinline__ int read_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ int64_t read_lane(int64_t x, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(uint32_t(uint64_t(x)), lane), hi = __builtin_amdgcn_readlane(uint32_t(uint64_t(x) >> 32), lane);
    return int64_t(uint64_t(hi) << 32 | lo);
}
// Over a wavefront: the maximum of values that are not negative.
__device__ __forceinline__ int wave_maximum(int x) {
    wave_prefix([&](auto ctrl, auto rows) { x = max(x, before<decltype(ctrl)::value, decltype(rows)::value>(x)); });
    return read_lane(x, kWaveSize - 1);
}
// a / b for 0 <= a, 0 < b, a / b < 2^40: by way of float64 and a reciprocal that is good to some 2^-48, so that the quotient is
// off by one at most (the compiler's division takes many times the instructions, and those are what a small call waits for).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    double r = __builtin_amdgcn_rcp(double(b));
    r = fma(fma(-double(b), r, 1.0), r, r);
    int64_t q = int64_t(double(a) * r);
    const int64_t left = a - q * b;
    if (left < 0) --q;
    if (left >= b) ++q;
    return q;
}

// The sequences as a wavefront holds them: a lane stands for `per_lane` consecutive ones.
struct Sequences {
    const PagedStep& s;
    int positions;      // rows of a block
    double inverse;     // 1 / positions
    int per_lane;
    Sequence own;       // the first of this lane's
    __device__ __forceinline__ Sequence sequence(int b) const {
        const int from = s.q_offsets[b], to = s.q_offsets[b + 1], len = s.kv_lens[b];
        Sequence q;
        q.row = min(max(from, 0), s.rows);
        q.n = max(min(to, s.rows) - q.row, 0);
        q.kv = min(max(len, 0), s.max_kv);
        q.blocks = blocks_up_to(q.n);
        q.falls = to < from;
        return q;
    }
    // Blocks whose rows are all among the first n: n / positions (the half keeps the product off the whole numbers).
    __device__ __forceinline__ int whole_blocks(int n) const { return int((double(n) + 0.5) * inverse); }
    __device__ __forceinline__ int blocks_up_to(int n) const { return int((double(uint32_t(n + positions - 1)) + 0.5) * inverse); }
    // Blocks of `columns` (1, 2, 4 or 8) times the positions of 16 columns.
    __device__ __forceinline__ Sequences(const PagedAttnParams& p, int columns)
        : s(p.step), positions(columns * p.positions), inverse(p.per_position / columns), per_lane((p.step.seqs + kWaveSize - 1) / kWaveSize) {
        const int b = int(threadIdx.x & (kWaveSize - 1)) * per_lane;
        own = sequence(min(b, s.seqs - 1));
        if (b >= s.seqs) own.n = own.blocks = 0;
    }
    // The same sequences in blocks of half the size.
    __device__ __forceinline__ void halve() {
        positions /= 2;
        inverse *= 2.0;
        own.blocks = blocks_up_to(own.n);
    }
    // of(sequence) for every sequence of this lane
    template <typename F>
    __device__ __forceinline__ void each(F of) const {
        of(own);
        const int b = int(threadIdx.x & (kWaveSize - 1)) * per_lane;
        for (int i = 1; i < per_lane; ++i) {
            if (b + i < s.seqs) of(sequence(b + i));
        }
    }
    __device__ __forceinline__ Sequence at(int b) const {   // b is uniform
        if (per_lane == 1) return {read_lane(own.row, b), read_lane(own.n, b), read_lane(own.kv, b), read_lane(own.blocks, b), false};
        const Sequence q = sequence(b);
        return {wave_uniform(q.row), wave_uniform(q.n), wave_uniform(q.kv), wave_uniform(q.blocks), false};
    }
};

// A sum over all sequences, and the sequence at a place of it.  of(sequence): a sequence's addend.
template <typename T, typename F>
struct Shares {
    const Sequences& all;
    const F of;
    T upto, total;   // up to and with this lane's sequences (in every lane its own), all
    __device__ __forceinline__ Shares(const Sequences& sequences, F f) : all(sequences), of(f) {
        T mine = 0;
        all.each([&](const Sequence& q) { mine += of(q); });
        upto = wave_scan(mine);
        total = read_lane(upto, kWaveSize - 1);
    }
    // The sequence in whose addend place x (0 <= x < total) lies; x becomes the place in it.
    __device__ __forceinline__ int find(T& x) const {
        const int lane = threadIdx.x & (kWaveSize - 1);
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x) | uint64_t(1) << 63);
        if (at > 0) x -= read_lane(upto, at - 1);
        if (all.per_lane == 1) return min(at, all.s.seqs - 1);
        const int end = min((at + 1) * all.per_lane, all.s.seqs);
        for (int base = at * all.per_lane; base < end; base += kWaveSize) {
            const T sum = wave_scan(base + lane < end ? of(all.sequence(base + lane)) : T(0));
            const uint64_t here = __builtin_amdgcn_ballot_w64(sum > x);
            if (here) {
                const int i = __builtin_ctzll(here);
                if (i > 0) x -= read_lane(sum, i - 1);
                return base + i;
            }
            x -= read_lane(sum, kWaveSize - 1);
        }
        return all.s.seqs - 1;   // (the addends are those of the sum: one of the loop's steps has returned)
    }
};

// Keys and values of one sequence and kv head.
//
// A wavefront-wide load takes G consecutive token rows, which lie in one page.  Its address is a scalar; those of a wavefront's
// next 64 loads are worked out side by side, lane i for load i (a page number per lane, fetched 64 loads ahead), and read
// from there.  A load that would begin behind the last token takes the last token's rows again, and rows behind the last token
// are read as they lie in its page: whatever is there is hidden from every column.
struct PagedHead {
    const char *k, *v;         // the head's dims in page 0
    int64_t k_page, v_page;    // bytes
    int k_pitch, v_pitch;      // bytes from a token to the next (below 2^25)
    const int* table;          // the sequence's pages
    int shift, last_page;      // pages of the cache - 1
    int last;                  // last token
    // The page of this lane's load, whose first token is `token`.
    __device__ __forceinline__ int page_of(int token) const { return table[min(token, last) >> shift]; }
    // Its address.
    __device__ __forceinline__ void rows_at(int page, int token, int G, int64_t& kp, int64_t& vp) const {
        const int in = min(token, last) & ((1 << shift) - 1) & ~(G - 1);
        page = min(max(page, 0), last_page);
        kp = reinterpret_cast<int64_t>(k) + page * k_page + int64_t(in) * k_pitch;
        vp = reinterpret_cast<int64_t>(v) + page * v_page + int64_t(in) * v_pitch;
    }
};

// Values that are not finite, in tiles that hold tokens which some column does not see.  0 times infinity is not 0, so there
// they are taken out of V before the product, and the block remembers for every dim the first token at which one was taken
// out; the columns that see that token get it back at the end.
template <int HD>
struct OddValues {
    int up[HD], down[HD];   // first token with +infinity or NaN, with -infinity or NaN
    int any;
    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < HD; i += kThreads) up[i] = down[i] = 0x7fffffff;
        if (threadIdx.x == 0) any = 0;
    }
    static __device__ __forceinline__ uint32_t is_odd(uint32_t x) { return uint32_t((x & 0x7f80u) == 0x7f80u) | uint32_t((x & 0x7f800000u) == 0x7f800000u); }
    static __device__ __forceinline__ uint32_t is_odd(const uint4& v) { return is_odd(v.x) | is_odd(v.y) | is_odd(v.z) | is_odd(v.w); }
    // Takes what is not finite out of a token's eight values from dim on, which lie in LDS.
    __device__ __forceinline__ void take_out(unsigned char* at, int token, int dim) {
        uint16_t* const v = reinterpret_cast<uint16_t*>(at);
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = v[i];
            if ((x & 0x7f80u) != 0x7f80u) continue;
            const bool nan = (x & 0x7fu) != 0;
            if (nan || !(x & 0x8000u)) atomicMin(&up[dim + i], token);
            if (nan || (x & 0x8000u)) atomicMin(&down[dim + i], token);
            v[i] = 0;
            any = 1;
        }
    }
    // What a column that sees the tokens below `limit` has of dim `dim` and the next three.
    __device__ __forceinline__ f32x4_t seen(f32x4_t o, int dim, int limit) const {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (up[dim + r] < limit) o[r] += __builtin_inff();
            if (down[dim + r] < limit) o[r] -= __builtin_inff();
        }
        return o;
    }
};

// Sum over the four k groups of a column (lanes l, l ^ 16, l ^ 32, l ^ 48), in every one of them.
__device__ __forceinline__ float column_sum(float x) {
    const uint32_t xi = __builtin_bit_cast(uint32_t, x);
    const auto h = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
    const float y = __builtin_bit_cast(float, uint32_t(h[0])) + __builtin_bit_cast(float, uint32_t(h[1]));
    const uint32_t yi = __builtin_bit_cast(uint32_t, y);
    const auto r = __builtin_amdgcn_permlane16_swap(yi, yi, false, false);
    return __builtin_bit_cast(float, uint32_t(r[0])) + __builtin_bit_cast(float, uint32_t(r[1]));
}

// The softmax state of 16 columns: O[nb][r] is dim 16 nb + 4 fg + r of column fn.
template <int HD>
struct Columns {
    f32x4_t O[HD / 16];
    float m, l;   // l: this lane's share (of the four k groups)
};

// ------------------------------------------------------------------------------------------------------------- narrow
// First token of this lane's load: the lanes stand for the loads of the tiles t, t + step, ...
template <int HD, int LOADS>
__device__ __forceinline__ int narrow_token(int t, int step) {
    const int lane = threadIdx.x & (kWaveSize - 1);
    return t + lane / LOADS * step + lane % LOADS * MfmaTile<HD, LOADS>::G;
}
// A wavefront's tiles t, t + step, ... < t_stop of a narrow block, through its own slab, as in the dense kernels: the next
// tile's loads go out as soon as this one's registers are in the slab.
template <int HD, int LOADS, int CB>
__device__ __forceinline__ void narrow_tiles(const PagedHead& h, unsigned char* slab, const bf16x8_t (&q)[CB][HD / 32], int page, int page_next, int t,
                                             int t_stop, int step, const int (&limit)[CB], int limit_min, float c, Columns<HD> (&col)[CB],
                                             OddValues<HD>& odd) {
    using T = MfmaTile<HD, LOADS>;
    constexpr int LPR = T::LPR, G = T::G, U = T::U, WT = T::WT, NG = T::NG, KC = T::KC, NB = T::NB, KS = T::KS;
    constexpr int KPITCH = T::KPITCH, VPITCH = T::VPITCH;
    if (t >= t_stop) return;
    const int lane = threadIdx.x & (kWaveSize - 1);
    const int ld_row = lane / LPR, ld_c = lane % LPR, fg = lane >> 4;
    unsigned char* wr_k = slab + ld_row * KPITCH + ld_c * 16;
    unsigned char* wr_v = slab + ld_row * VPITCH + ld_c * 16;
    const unsigned char* rd_k = slab + (lane & 15) * KPITCH + fg * 16;
    const unsigned char* rd_v = slab + (4 * fg + ((lane & 15) >> 2)) * VPITCH + (lane & 3) * 8;
    const uint32_t k_off = uint32_t(ld_row) * uint32_t(h.k_pitch) + uint32_t(ld_c) * 16u, v_off = uint32_t(ld_row) * uint32_t(h.v_pitch) + uint32_t(ld_c) * 16u;

    uint4 kr[U], vr[U];
    auto load = [&](uint4 (&dst)[U], int64_t rows, int first, uint32_t off) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) dst[u] = load16_stream(reinterpret_cast<const uint16_t*>(read_lane(rows, first + u) + off));
    };
    constexpr int AHEAD = kWaveSize / U;   // tiles whose loads the lanes hold
    int token = narrow_token<HD, LOADS>(t, step), first = 0;
    int64_t k_rows, v_rows;
    h.rows_at(page, token, G, k_rows, v_rows);
    load(kr, k_rows, 0, k_off);
    load(vr, v_rows, 0, v_off);
    for (; t < t_stop; t += step) {
        const int tn = t + step;
        const bool more = tn < t_stop;
#pragma unroll
        for (int u = 0; u < U; ++u) *reinterpret_cast<uint4*>(wr_k + u * G * KPITCH) = kr[u];
        lds_phase_fence();
        if (more) {
            first += U;
            if (first == kWaveSize) {
                first = 0;
                token += AHEAD * step;
                h.rows_at(page_next, token, G, k_rows, v_rows);
                page_next = h.page_of(token + AHEAD * step);
            }
            load(kr, k_rows, first, k_off);
        }

        u32x4_t a[NG * KC];
#pragma unroll
        for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
            for (int m = 0; m < KC; ++m) a[tg * KC + m] = *reinterpret_cast<const u32x4_t*>(rd_k + tg * 16 * KPITCH + m * 64);
        }
        if constexpr (CB == 1) pin_all(a);
        f32x4_t S[CB][NG];
#pragma unroll
        for (int m = 0; m < KC; ++m) {
#pragma unroll
            for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    S[cb][tg] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a[tg * KC + m]), q[cb][m],
                                                                        m == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : S[cb][tg], 0, 0, 0);
                }
            }
        }
        lds_phase_fence();
        const bool hidden = t + WT > limit_min;   // some column does not see some token
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            if (hidden) {
                const int visible = limit[cb] - t - 4 * fg;
#pragma unroll
                for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (tg * 16 + j >= visible) S[cb][tg][j] = -__builtin_inff();
                    }
                }
            }
            float top = S[cb][0][0];
#pragma unroll
            for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
                for (int j = 0; j < 4; ++j) top = maximum(top, S[cb][tg][j]);
            }
            top = column_maximum(top);
            if (__builtin_amdgcn_ballot_w64(top > col[cb].m) != 0) {
                const float m_new = fmaxf(col[cb].m, top);
                const float alpha = fast_exp2((col[cb].m - m_new) * c);
                col[cb].l *= alpha;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) col[cb].O[nb] *= alpha;
                col[cb].m = m_new;
            }
            const float mc = col[cb].m * c;
            float sum = 0.f;
#pragma unroll
            for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    S[cb][tg][j] = fast_exp2(fmaf(S[cb][tg][j], c, -mc));
                    sum += S[cb][tg][j];
                }
            }
            col[cb].l += sum;
        }

#pragma unroll
        for (int u = 0; u < U; ++u) *reinterpret_cast<uint4*>(wr_v + u * G * VPITCH) = vr[u];
        lds_phase_fence();
        if (hidden) {
            uint32_t found = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) found |= odd.is_odd(vr[u]);
            if (__builtin_amdgcn_ballot_w64(found) != 0) {
#pragma unroll 1
                for (int u = 0; u < U; ++u) odd.take_out(wr_v + u * G * VPITCH, t + u * G + ld_row, ld_c * 8);
            }
            lds_phase_fence();
        }
        if (more) load(vr, v_rows, first, v_off);

        s16x4_t vt[KS * NB * 2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    vt[(ks * NB + nb) * 2 + half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        L3_LDS_PTR(s16x4_t, rd_v + (2 * ks + half) * 16 * VPITCH + nb * 32));
                }
            }
        }
        if constexpr (CB == 1) pin_all(vt);   // (two column blocks have no registers for it: 48.5 us instead of 43.6 for drafted tokens)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            bf16x8_t p[CB];
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const f32x4_t &lo = S[cb][2 * ks], &hi = S[cb][2 * ks + 1];
                p[cb] = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]),
                                                                pack_bf16x2(hi[2], hi[3])));
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const s16x8_t v = __builtin_shufflevector(vt[(ks * NB + nb) * 2], vt[(ks * NB + nb) * 2 + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    col[cb].O[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), p[cb], col[cb].O[nb], 0, 0, 0);
                }
            }
        }
        lds_phase_fence();
    }
}

// --------------------------------------------------------------------------------------------------------------- wide
template <int HD>
struct WideTile {
    static constexpr int NG = kTile / 16, KS = kTile / 32, KC = HD / 32, NB = HD / 16;
    static constexpr int CPR = HD / 8, ROWB = HD * 2, KBYTES = kTile * ROWB, STAGE = 2 * KBYTES;
    static constexpr int G = kWaveSize / CPR;                       // token rows of a wavefront-wide load
    static constexpr int IPW = kTile / G / kWaves;                  // loads of K (and of V) per wavefront
    static constexpr __host__ __device__ int key(int row) { return HD == 128 ? (row & 15) : ((row >> 1) & 7); }
};

// A wavefront's share of a wide block: two column blocks, and what one tile on its LDS stage does to them.
// The softmax denominator rides on the matrix pipe (a block of ones as one more row block of V^T), so that the weights that
// are added up are those that are multiplied.
template <int HD, int CB>
struct WideWave {
    using T = WideTile<HD>;
    static constexpr int NG = T::NG, KS = T::KS, KC = T::KC, NB = T::NB, ROWB = T::ROWB;
    bf16x8_t q[CB][KC];
    f32x4_t O[CB][NB];
    float m[CB], l[CB];  // reference of the exponentials, denominator
    int limit[CB];       // a column sees the tokens below it
    int limit_min, stop; // of the wavefront: tiles below limit_min need no mask, tiles from stop on are skipped
    int ak[KC], av[NB];  // operand addresses in a stage
    bf16x8_t ones;

    __device__ __forceinline__ void addresses() {
        const int lane = threadIdx.x & (kWaveSize - 1), fn = lane & 15, fg = lane >> 4;
#pragma unroll
        for (int i = 0; i < KC; ++i) ak[i] = fn * ROWB + (((i * 4 + fg) ^ T::key(fn)) << 4);
        const int row = 4 * fg + (fn >> 2);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) av[nb] = T::KBYTES + row * ROWB + (((nb * 2 + ((lane & 3) >> 1)) ^ T::key(row)) << 4) + (lane & 1) * 8;
        ones = __builtin_bit_cast(bf16x8_t, make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
        asm volatile("" : "+v"(ones));
    }

    __device__ __forceinline__ uint4 k_operand(const unsigned char* stage, int tg, int i) const {
        return *reinterpret_cast<const uint4*>(stage + ak[i] + tg * 16 * ROWB);
    }
    __device__ __forceinline__ s16x8_t v_operand(const unsigned char* stage, int ks, int nb) const {
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(L3_LDS_PTR(s16x4_t, stage + av[nb] + (2 * ks) * 16 * ROWB));
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(L3_LDS_PTR(s16x4_t, stage + av[nb] + (2 * ks + 1) * 16 * ROWB));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ f32x4_t product(const uint4& a, const bf16x8_t& b, const f32x4_t& acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), b, acc, 0, 0, 0);
    }
    __device__ __forceinline__ void hide(f32x4_t (&S)[NG], int cb, int t0) const {
        const int visible = limit[cb] - t0 - 4 * ((threadIdx.x & (kWaveSize - 1)) >> 4);
#pragma unroll
        for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (tg * 16 + j >= visible) S[tg][j] = -__builtin_inff();
            }
        }
    }
    // The reference of column block cb moves up to the largest of its scores (by `slack` at least), O and l with it.
    __device__ __forceinline__ void raise(const f32x4_t (&S)[NG], int cb, float slack, float c) {
        float top = S[0][0];
#pragma unroll
        for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
            for (int j = 0; j < 4; ++j) top = maximum(top, S[tg][j]);
        }
        top = column_maximum(top);
        if (__builtin_amdgcn_ballot_w64(top > m[cb] + slack) != 0) {
            const float m_new = fmaxf(m[cb], top);
            const float alpha = fast_exp2((m[cb] - m_new) * c);
            l[cb] *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) O[cb][nb] *= alpha;
            m[cb] = m_new;
        }
    }
    // Weights of column block cb against its reference, and their sum over the tile (in every lane its column's).
    __device__ __forceinline__ float weights(f32x4_t (&S)[NG], int cb, float c, bf16x8_t (&p)[KS]) const {
        const float mc = m[cb] * c;
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
            for (int j = 0; j < 4; ++j) S[tg][j] = fast_exp2(fmaf(S[tg][j], c, -mc));
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            p[ks] = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(S[2 * ks][0], S[2 * ks][1]), pack_bf16x2(S[2 * ks][2], S[2 * ks][3]),
                                                            pack_bf16x2(S[2 * ks + 1][0], S[2 * ks + 1][1]),
                                                            pack_bf16x2(S[2 * ks + 1][2], S[2 * ks + 1][3])));
            sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[ks], sum, 0, 0, 0);
        }
        return sum[0];
    }

    // The tile in the compiler's order: scores, maximum, weights, product.  The reference follows the scores only where one
    // exceeds it by 2^8 (weights stay below 256, which bf16 and the float32 sums hold as well as those below 1).
    __device__ __forceinline__ void tile(const unsigned char* stage, int t0, float c) {
        f32x4_t S[CB][NG];
#pragma unroll
        for (int tg = 0; tg < NG; ++tg) {
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const uint4 a = k_operand(stage, tg, i);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) S[cb][tg] = product(a, q[cb][i], i == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : S[cb][tg]);
            }
        }
        const bool hidden = t0 + kTile > limit_min;
        bf16x8_t p[CB][KS];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            if (hidden) hide(S[cb], cb, t0);
            raise(S[cb], cb, 8.0f / c, c);
            l[cb] += weights(S[cb], cb, c, p[cb]);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const uint4 v = __builtin_bit_cast(uint4, v_operand(stage, ks, nb));
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) O[cb][nb] = product(v, p[cb][ks], O[cb][nb]);
            }
        }
    }

    // The same laid out by hand, 32 tokens at a time, for wavefronts with the registers of two per SIMD: the vector work of one
    // column block is issued between the matrix instructions of the other, operands are requested a phase ahead.
    //   S0 = K Q0^T
    //   [S1 = K Q1^T        | exponentials of S0]     V^T operands requested half way
    //   [O0^T += V^T P0     | exponentials of S1]     the next 32 tokens' K operands requested in front
    //    O1^T += V^T P1
    // No maximum in the common case: the weights are taken against the reference as it stands, and their sum, which the
    // matrix pipe forms anyway, says whether that was safe (at most 1024: every weight was).  If not -- the first tile, a
    // score that leaves the reference far behind, a NaN -- the block's scores are formed again and the reference raised.
    __device__ __forceinline__ void tile_by_hand(const unsigned char* stage, int t0, float c) {
        constexpr int G2 = 2, NQ = KC * G2, NP = NB, NS = G2 * 4;   // 16-token groups; matrix instructions of scores and of output; scores per lane
        static_assert(CB == 2, "two column blocks take turns");
        constexpr float kSumLimit = 1024.0f;
        const f32x4_t none = {0.f, 0.f, 0.f, 0.f};
        uint4 k[G2][KC];
        auto request_k = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < KC; ++i) {
#pragma unroll
                for (int tg = 0; tg < G2; ++tg) k[tg][i] = k_operand(stage, 2 * ks + tg, i);
            }
        };
        request_k(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bool hidden = t0 + 32 * (ks + 1) > limit_min;
            f32x4_t S[CB][G2];
            uint32_t w[CB][NS / 2];
            bf16x8_t p[CB];
            s16x8_t v[NB];
            auto scores = [&](int cb) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < KC; ++i) {
#pragma unroll
                    for (int tg = 0; tg < G2; ++tg) S[cb][tg] = product(k[tg][i], q[cb][i], i == 0 ? none : S[cb][tg]);
                }
            };
            auto hide32 = [&](int cb) __attribute__((always_inline)) {
                if (hidden) {
                    const int visible = limit[cb] - t0 - 32 * ks - 4 * ((threadIdx.x & (kWaveSize - 1)) >> 4);
#pragma unroll
                    for (int tg = 0; tg < G2; ++tg) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (tg * 16 + j >= visible) S[cb][tg][j] = -__builtin_inff();
                        }
                    }
                }
            };
            auto score = [&](int cb, int i, float mc) __attribute__((always_inline)) {
                const int tg = i / 4, j = i % 4;
                S[cb][tg][j] = fast_exp2(fmaf(S[cb][tg][j], c, -mc));
                if (j & 1) w[cb][i / 2] = pack_bf16x2(S[cb][tg][j - 1], S[cb][tg][j]);
            };
            auto collect = [&](int cb) __attribute__((always_inline)) {
                p[cb] = __builtin_bit_cast(bf16x8_t, make_uint4(w[cb][0], w[cb][1], w[cb][2], w[cb][3]));
                float sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[cb], none, 0, 0, 0)[0];
                if (__builtin_amdgcn_ballot_w64(!(sum <= kSumLimit)) != 0) {
#pragma unroll
                    for (int i = 0; i < KC; ++i) {
#pragma unroll
                        for (int tg = 0; tg < G2; ++tg) S[cb][tg] = product(k_operand(stage, 2 * ks + tg, i), q[cb][i], i == 0 ? none : S[cb][tg]);
                    }
                    hide32(cb);
                    float top = S[cb][0][0];
#pragma unroll
                    for (int i = 1; i < NS; ++i) top = maximum(top, S[cb][i / 4][i % 4]);
                    const float m_new = fmaxf(m[cb], column_maximum(top)), alpha = fast_exp2((m[cb] - m_new) * c);
                    l[cb] *= alpha;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) O[cb][nb] *= alpha;
                    m[cb] = m_new;
#pragma unroll
                    for (int i = 0; i < NS; ++i) score(cb, i, m_new * c);
                    p[cb] = __builtin_bit_cast(bf16x8_t, make_uint4(w[cb][0], w[cb][1], w[cb][2], w[cb][3]));
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[cb], none, 0, 0, 0)[0];
                }
                l[cb] += sum;
            };
            __builtin_amdgcn_sched_barrier(0);
            scores(0);
            __builtin_amdgcn_sched_barrier(0);
            hide32(0);
            const float mc0 = m[0] * c;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int i = n / G2, tg = n % G2;
                S[1][tg] = product(k[tg][i], q[1][i], i == 0 ? none : S[1][tg]);
#pragma unroll
                for (int e = n * NS / NQ; e < (n + 1) * NS / NQ; ++e) score(0, e, mc0);
                __builtin_amdgcn_sched_barrier(0);
                if (n == NQ / 2 - 1) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) v[nb] = v_operand(stage, ks, nb);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            hide32(1);
            const float mc1 = m[1] * c;
            collect(0);
            __builtin_amdgcn_sched_barrier(0);
            if (ks + 1 < KS) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) asm volatile("" : "+v"(v[nb]));   // the wait for these precedes the next requests
                request_k(ks + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                O[0][n] = product(__builtin_bit_cast(uint4, v[n]), p[0], O[0][n]);
#pragma unroll
                for (int e = n * NS / NP; e < (n + 1) * NS / NP; ++e) score(1, e, mc1);
                __builtin_amdgcn_sched_barrier(0);
            }
            collect(1);
#pragma unroll
            for (int n = 0; n < NP; ++n) O[1][n] = product(__builtin_bit_cast(uint4, v[n]), p[1], O[1][n]);
        }
    }
};

__device__ __forceinline__ PagedHead head_of(const PagedAttnParams& p, int kv, int b, int kvh) {
    PagedHead h;
    h.k = reinterpret_cast<const char*>(p.k + kvh * p.k_sh);
    h.v = reinterpret_cast<const char*>(p.v + kvh * p.v_sh);
    h.k_page = p.k_sp * 2; h.v_page = p.v_sp * 2;
    h.k_pitch = int(p.k_st) * 2; h.v_pitch = int(p.v_st) * 2;
    h.table = p.step.table + b * p.step.table_stride;
    h.shift = p.step.page_shift;
    h.last_page = p.step.pages - 1;
    h.last = kv - 1;
    return h;
}

// Dims (4 m + fg) 8 ... of a column's query row for every m: the right operand of the scores.
template <int HD>
__device__ __forceinline__ void load_query(const PagedAttnParams& p, int64_t row, int h, bool valid, bf16x8_t (&q)[HD / 32]) {
    const int fg = (threadIdx.x & (kWaveSize - 1)) >> 4;
#pragma unroll
    for (int m = 0; m < HD / 32; ++m) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (valid) v = load16(p.q + row * p.q_sr + h * p.q_sh + (m * 4 + fg) * 8);
        q[m] = __builtin_bit_cast(bf16x8_t, v);
    }
}

// One wide block, or a piece of its tokens, by a workgroup: tokens t_first .. t_stop - 1 (whole tiles, but for the block's
// last).  `slot`: where a piece leaves its state, null: the block is whole.
template <int HD, int CB, int WPE>
__device__ __forceinline__ void wide_block(const PagedAttnParams& p, const PagedHead& h, int kvh, int row, int rows, int first_pos, int t_first,
                                           int t_stop, char* slot, int units, unsigned char* s_stage0, unsigned char* s_stage1, OddValues<HD>& odd) {
    using W = WideTile<HD>;
    constexpr int NB = HD / 16;
    const int tid = threadIdx.x, lane = tid & (kWaveSize - 1), wave = wave_uniform(tid / kWaveSize), fn = lane & 15, fg = lane >> 4;
    const int ld_row = lane / W::CPR, wave_row = wave * W::IPW * W::G;   // of the wavefront's loads, below
    // the lanes stand for the loads of the next AHEAD tiles; what else there is to do before the first load waits for the pages
    constexpr int AHEAD = kWaveSize / W::IPW;
    int token = t_first + lane / W::IPW * kTile + wave_row + lane % W::IPW * W::G, page = 0, page_next = 0;
    if (t_first < t_stop) {
        page = h.page_of(token);
        page_next = h.page_of(token + AHEAD * kTile);
    }
    const float c = p.scale_log2e;
    const int turn = int(blockIdx.x) / units;
    WideWave<HD, CB> ww;
    const int wave_pos = wave * CB * p.positions;     // of the wavefront's first column
    const int wave_rows = min(rows - wave_pos, CB * p.positions);
    ww.stop = wave_rows > 0 ? min(t_stop, first_pos + wave_pos + wave_rows) : 0;
    ww.limit_min = first_pos + wave_pos + 1;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int of = fn * p.inverse >> 8, i = wave_pos + cb * p.positions + of;
        const bool valid = of < p.positions && i < rows;
        ww.limit[cb] = valid ? first_pos + i + 1 : 0;
        load_query<HD>(p, row + i, kvh * p.R + fn - of * p.R, valid, ww.q[cb]);
    }
    // global -> LDS: load i of the wavefront has token rows (wave IPW + i) G ... of the tile; the 16-byte chunk c of row r lies
    // at position c ^ key(r).
    int chunk0 = ((lane % W::CPR) ^ W::key(ld_row)) * 16;   // of load 0; of load i: its third bit from above turned i times
    uint32_t k_row = uint32_t(ld_row) * uint32_t(h.k_pitch), v_row = uint32_t(ld_row) * uint32_t(h.v_pitch);
    static_assert(W::key(W::G) == 4 && (W::IPW <= 2 || W::key(3 * W::G) == 12), "the keys of a load's rows are four further than the load's before");
    int64_t k_rows, v_rows;
    h.rows_at(page, token, W::G, k_rows, v_rows);
    int first = 0;   // lane of the next tile's first load
    auto dma = [&](unsigned char* stage) __attribute__((always_inline)) {
        asm volatile("" : "+v"(chunk0), "+v"(k_row), "+v"(v_row));   // (sums of these are not worth registers across the tile)
#pragma unroll
        for (int i = 0; i < W::IPW; ++i) {
            const int inst = wave * W::IPW + i;
            const int chunk = chunk0 ^ (i << 6);
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(read_lane(k_rows, first + i)), 0, -1, 0x00020000);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(read_lane(v_rows, first + i)), 0, -1, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, L3_LDS_PTR(void, stage + inst * 1024), 16, int(k_row) + chunk, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, L3_LDS_PTR(void, stage + W::KBYTES + inst * 1024), 16, int(v_row) + chunk, 0, 0, 0);
        }
        first += W::IPW;
        if (first == kWaveSize) {
            first = 0;
            token += AHEAD * kTile;
            h.rows_at(page_next, token, W::G, k_rows, v_rows);
            page_next = h.page_of(token + AHEAD * kTile);
        }
    };
    // Until this wavefront's part of a stage has landed; what is not finite is taken out of a V tile with hidden tokens by
    // the lane that loaded it.
    auto landed = [&](int t0, unsigned char* stage) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0xF70);   // vmcnt(0)
        if (t0 + kTile > first_pos + 1 && t0 < t_stop) {   // workgroup-uniform
#pragma unroll 1
            for (int i = 0; i < W::IPW; ++i) {
                const int inst = wave * W::IPW + i, r = inst * W::G + ld_row;
                unsigned char* const at = stage + W::KBYTES + inst * 1024 + lane * 16;
                if (odd.is_odd(*reinterpret_cast<const uint4*>(at))) odd.take_out(at, t0 + r, ((lane % W::CPR) ^ W::key(r)) * 8);
            }
        }
        __syncthreads();
    };
    if (t_first < t_stop) dma(s_stage0);
    ww.addresses();
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        ww.m[cb] = kNothing;
        ww.l[cb] = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) ww.O[cb][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    if (t_first < t_stop) {
        landed(t_first, s_stage0);
        auto step = [&](auto parity, int t0) __attribute__((always_inline)) {
            constexpr bool ODD = decltype(parity)::value;
            if (t0 + kTile < t_stop) dma(ODD ? s_stage0 : s_stage1);   // workgroup-uniform
            // The oldest wavefront of a SIMD goes first, so of two workgroups of one length the older ends at 1.8 us a tile and
            // leaves the other, at 2.3, alone with the compute unit.  They take turns instead.
            if ((t0 / kTile ^ turn) & 1) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            if (t0 < ww.stop) {
                const unsigned char* const stage = ODD ? s_stage1 : s_stage0;
                if constexpr (CB == 2 && WPE <= 2) ww.tile_by_hand(stage, t0, c);
                else ww.tile(stage, t0, c);
            }
            landed(t0 + kTile, ODD ? s_stage0 : s_stage1);
        };
        for (int t0 = t_first; t0 < t_stop; t0 += 2 * kTile) {
            step(std::false_type{}, t0);
            if (t0 + kTile < t_stop) step(std::true_type{}, t0 + kTile);
        }
    }
    // (places in the output are worked out again here: kept across the tiles they would cost registers that the tiles need)
    int fn2 = fn, pos2 = wave_pos;
    asm volatile("" : "+v"(fn2), "+s"(pos2));
    const int of = fn2 * p.inverse >> 8;
    if (odd.any) {   // written before the last barrier; this is the workgroup's only block
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) ww.O[cb][nb] = odd.seen(ww.O[cb][nb], nb * 16 + fg * 4, ww.limit[cb]);
        }
    }
    if (!slot) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            const int i = pos2 + cb * p.positions + of;
            if (of < p.positions && i < rows) {
                const float inv = ww.limit[cb] > 0 ? 1.0f / ww.l[cb] : 0.f;
                uint16_t* const o = p.out + int64_t(row + i) * p.o_sr + (kvh * p.R + fn2 - of * p.R) * p.o_sh + fg * 4;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    *reinterpret_cast<uint2*>(o + nb * 16) = make_uint2(pack_bf16x2(ww.O[cb][nb][0] * inv, ww.O[cb][nb][1] * inv),
                                                                        pack_bf16x2(ww.O[cb][nb][2] * inv, ww.O[cb][nb][3] * inv));
                }
            }
        }
    } else if (pos2 < rows) {   // as it lies in the registers, so that every access is whole lines
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) *reinterpret_cast<f32x4_t*>(slot + ((cb * NB + nb) * kThreads + tid) * 16) = ww.O[cb][nb];
            *reinterpret_cast<float2*>(slot + CB * NB * kThreads * 16 + (cb * kThreads + tid) * 8) = make_float2(ww.m[cb], ww.l[cb]);
        }
    }
}

// One narrow block, or a piece of its tokens.
template <int HD, int LOADS, int CB>
struct NarrowArea {   // LDS of a wavefront: its slab, and later its state
    static constexpr int OPITCH = HD * 4 + 16;
    static constexpr int COLUMNS = CB * 16 * OPITCH;
    static constexpr int BYTES = std::max(MfmaTile<HD, LOADS>::SLAB, COLUMNS + CB * 128);
};
template <int HD, int LOADS, int CB>
__device__ __forceinline__ void narrow_block(const PagedAttnParams& p, const PagedHead& h, int kvh, int row, int rows, int first_pos, int t_first,
                                             int t_stop, char* slot, unsigned char* s_mem, OddValues<HD>& odd) {
    using N = MfmaTile<HD, LOADS>;
    using A = NarrowArea<HD, LOADS, CB>;
    constexpr int NB = HD / 16;
    const int tid = threadIdx.x, lane = tid & (kWaveSize - 1), wave = wave_uniform(tid / kWaveSize), fn = lane & 15, fg = lane >> 4;
    const float c = p.scale_log2e;
    const int t = t_first + wave * N::WT;
    int page = 0, page_next = 0;   // what else there is to do before the first load waits for them
    if (t < t_stop) {
        const int token = narrow_token<HD, LOADS>(t, kWaves * N::WT);
        page = h.page_of(token);
        page_next = h.page_of(token + kWaveSize / LOADS * kWaves * N::WT);
    }
    bf16x8_t q[CB][HD / 32];
    Columns<HD> col[CB];
    int limit[CB];   // a column sees the tokens below it
    const int of = fn * p.inverse >> 8;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int i = cb * p.positions + of;
        const bool valid = of < p.positions && i < rows;
        limit[cb] = valid ? first_pos + i + 1 : 0;
        load_query<HD>(p, row + i, kvh * p.R + fn - of * p.R, valid, q[cb]);
        col[cb].m = kNothing;
        col[cb].l = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) col[cb].O[nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    unsigned char* const mem = s_mem + wave * A::BYTES;
    narrow_tiles<HD, LOADS, CB>(h, mem, q, page, page_next, t, t_stop, kWaves * N::WT, limit, first_pos + 1, c, col, odd);
    // the four wavefronts' states meet in LDS, over the slabs
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const float l = column_sum(col[cb].l);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) *reinterpret_cast<f32x4_t*>(mem + (cb * 16 + fn) * A::OPITCH + nb * 64 + fg * 16) = col[cb].O[nb];
        if (fg == 0) *reinterpret_cast<float2*>(mem + A::COLUMNS + (cb * 16 + fn) * 8) = make_float2(col[cb].m, l);
    }
    __syncthreads();
    const int oc = tid / 16, od = tid % 16, oof = oc * p.inverse >> 8;   // this thread: column of each block, and dims od * (HD / 16) ...
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        const int i = cb * p.positions + oof, column = cb * 16 + oc;
        if (oof >= p.positions || i >= rows) continue;
        float2 ml[kWaves];
        float m = kNothing, sum = 0.f, o[NB];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            ml[w] = *reinterpret_cast<const float2*>(s_mem + w * A::BYTES + A::COLUMNS + column * 8);
            m = fmaxf(m, ml[w].x);
        }
#pragma unroll
        for (int e = 0; e < NB; ++e) o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = fast_exp2((ml[w].x - m) * c);
            sum = fmaf(ml[w].y, f, sum);
#pragma unroll
            for (int e = 0; e < NB; e += 4) {
                const f32x4_t part = *reinterpret_cast<const f32x4_t*>(s_mem + w * A::BYTES + column * A::OPITCH + (od * NB + e) * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e + r] = fmaf(part[r], f, o[e + r]);
            }
        }
        if (odd.any) {
#pragma unroll
            for (int e = 0; e < NB; e += 4) {
                const f32x4_t seen = odd.seen(f32x4_t{o[e], o[e + 1], o[e + 2], o[e + 3]}, od * NB + e, first_pos + i + 1);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e + r] = seen[r];
            }
        }
        if (!slot) {
            const float inv = first_pos + i >= 0 ? 1.0f / sum : 0.f;
            uint16_t* const out = p.out + int64_t(row + i) * p.o_sr + (kvh * p.R + oc - oof * p.R) * p.o_sh + od * NB;
#pragma unroll
            for (int e = 0; e < NB; e += 4) {
                *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16x2(o[e] * inv, o[e + 1] * inv), pack_bf16x2(o[e + 2] * inv, o[e + 3] * inv));
            }
        } else {
#pragma unroll
            for (int e = 0; e < NB; e += 4) {
                *reinterpret_cast<f32x4_t*>(slot + (column * HD + od * NB + e) * 4) = f32x4_t{o[e], o[e + 1], o[e + 2], o[e + 3]};
            }
            if (od == 0) *reinterpret_cast<float2*>(slot + CB * 16 * HD * 4 + column * 8) = make_float2(m, sum);
        }
    }
    const bool any = odd.any != 0;   // workgroup-uniform: written before the barrier above
    __syncthreads();   // before the slabs are written again
    if (any) {
        odd.clear();
        __syncthreads();
    }
}

// Rows of no sequence: zeros, by all workgroups together.
template <int HD>
__device__ __forceinline__ void clear_other_rows(const PagedAttnParams& p, int begin, int end) {
    for (int part = 0; part < 2; ++part) {
        const int from = part ? max(end, 0) : 0, to = part ? p.step.rows : min(begin, p.step.rows);
        for (int row = from + int(blockIdx.x); row < to; row += int(gridDim.x)) {
            for (int i = threadIdx.x; i < p.QH * (HD / 8); i += kThreads) {
                store16(p.out + row * p.o_sr + (i / (HD / 8)) * p.o_sh + (i % (HD / 8)) * 8, make_uint4(0u, 0u, 0u, 0u));
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ kernels
// How long wide blocks take, in us: a tile of a block that has its compute unit to itself (alone), and a tile's share of a unit
// that has as many as it can (full); with one and with two column blocks to a wavefront.  Measured with time stamps over one
// sequence, blocks of 4160 and more tokens.  What they decide is below: blocks of one or of two column blocks, and whether
// long blocks are cut.
template <int HD>
struct WideTime {
    static constexpr float alone1 = HD == 64 ? 0.70f : 1.05f, full1 = HD == 64 ? 0.30f : 0.66f;
    static constexpr float alone2 = HD == 64 ? 1.12f : 1.40f, full2 = HD == 64 ? 0.46f : 0.90f;
    static constexpr float start = 0.7f;   // of a workgroup, its share of a unit
    static constexpr float merge = 8.0f;   // the last launch, and partial results written
    // Pieces to a unit where blocks are cut: a choice between calls, none is best for all.  us with 2, 3 (taken), 4 at head size 64:
    // three prompts' pieces beside 13 generating sequences 67, 60, 67; two beside 30 of them 75, 68, 68; one beside 8 of 8000
    // tokens 44, 48, 44; 512 of 4096 tokens, 300 of 2500, 4 x 200 of 3000, 24 x 12 of 500 to 4000: within 1.  With 1, 2 (taken), 3 at
    // 128: three beside 13 98, 107, 97; 512 of 7012 tokens 99, 73, 92; 2 x 700 of 5000 144, 148, 149; 4 x 200 of 3000 66, 79, 74; 24 x 12 of
    // 500 to 4000 53, 56, 55.
    static constexpr int pieces = HD == 64 ? 3 : 2;
};

// What a workgroup of a wide launch does.
struct WideItem {
    int b, kvh, kv;          // sequence, kv head, tokens of the sequence
    int row, rows, first;    // the block: first row, rows (0: nothing to do, -1: no row is a sequence's), position of the first row
    int t_first, t_stop;     // its tokens, or the piece's
    int slot;                // of the piece's partial result; -1: the block is whole
    int two;                 // two column blocks to a wavefront, or one
};

// Finds it out; for one wavefront (all four at it would take four times the issue slots, and a launch's workgroups begin
// together).  2.5 to 4 us after a workgroup's start it is known: the arguments 0.6, the sequences 0.2, the choice 0.4, the search
// for the item 1 to 2.
template <int HD, int WPE>
__device__ __forceinline__ WideItem wide_item(const PagedAttnParams& p, const PagedGrid& grid) {
    using Time = WideTime<HD>;
    WideItem o;
    o.rows = 0;
    Sequences sequences(p, 2 * kWaves);

    // The longest block, and all blocks' tiles to a compute unit, in blocks of two column blocks (of one: about twice as many).
    auto tiles_of = [](int tokens) { return (tokens + kTile - 1) / kTile; };
    int longest = 0;
    float weight = 0.f, blocks = 0.f;
    bool falls = false;
    sequences.each([&](const Sequence& q) {
        falls |= q.falls;
        if (q.blocks > 0) {
            longest = max(longest, tiles_of(q.kv));
            blocks += float(q.blocks);
            weight += float(q.blocks) * (float(q.past()) + 0.5f * float(sequences.positions) * float(q.blocks + 1));
        }
    });
    // Only sequences that do not overlap have as many blocks as the launch has workgroups, and no piece without one.
    if (__builtin_amdgcn_ballot_w64(falls) != 0) {
        o.rows = -1;
        if (grid.entries > 0 && blockIdx.x == 0) grid.cuts[0].pieces = 0;
        return o;
    }
    longest = wave_maximum(longest);
    const float per_unit = wave_sum(weight) * float(p.KVH) / float(grid.units * kTile);
    const float blocks_per_unit = wave_sum(blocks) * float(p.KVH) / float(grid.units);
    const float uncut1 = fmaxf(float(longest) * Time::alone1, 2.f * (per_unit * Time::full1 + blocks_per_unit * Time::start));
    const float uncut2 = fmaxf(float(longest) * Time::alone2, per_unit * Time::full2 + blocks_per_unit * Time::start);
    const float cut2 = per_unit * Time::full2 + Time::merge;
    int most = kUncut;   // a block of more tiles is cut
    if (grid.entries > 0 && cut2 < fminf(uncut1, uncut2)) {
        most = max(int(fminf(per_unit * (1.05f / Time::pieces), 1e8f)) + 1, kLeastWidePiece);
        if (most >= longest) most = kUncut;
    }
    o.two = most < kUncut || uncut2 <= uncut1;
    if (!o.two) sequences.halve();
    const int positions = sequences.positions;

    // The items: blocks that are longer than most pieces, the pieces of those that are cut, the other blocks.  Blocks that are
    // whole go in order of their length.
    float per_piece = 1.0f / float(most);
    auto pieces_of = [&](int tiles) { return 1 + int(float(max(tiles - 1, 0)) * per_piece); };
    // first block of a sequence that has at least t tiles
    auto first_of = [&](const Sequence& q, int t) {
        const int below = kTile * (t - 1), d = below - (q.kv - q.n);   // tokens that are too few; rows that see no more than them
        return q.blocks == 0 ? 0 : q.kv <= below ? q.blocks : d < 0 ? 0 : min(sequences.whole_blocks(d), q.blocks - 1);
    };
    auto uncut_of = [&](const Sequence& q) { return most == kUncut ? q.blocks : first_of(q, most + 1); };
    auto pieces = [&](const Sequence& q) { return (q.blocks - uncut_of(q)) * pieces_of(tiles_of(q.kv)); };   // (as many as the longest has, for each)
    Shares<int, decltype(pieces)> cut(sequences, pieces);
    while (cut.total * int64_t(p.KVH) > grid.entries && most < kUncut) {   // more pieces than slots
        most = most + most / 2 >= longest ? kUncut : most + most / 2;
        per_piece = 1.0f / float(most);
        const Shares<int, decltype(pieces)> fewer(sequences, pieces);
        cut.upto = fewer.upto;
        cut.total = fewer.total;
    }
    const Shares<int, decltype(uncut_of)> whole(sequences, uncut_of);
    const int total = cut.total + whole.total;
    int item = int(blockIdx.x / unsigned(p.KVH));
    o.kvh = int(blockIdx.x) - item * p.KVH;
    if (grid.entries > 0 && blockIdx.x == 0) grid.cuts[0].pieces = cut.total * p.KVH;
    if (item >= total) return o;
    // Where the device holds all of them at once the dispatcher balances nothing: every second round over the compute units
    // is taken backwards, so that a unit has long and short ones.
    if (total * int64_t(p.KVH) <= WPE * grid.units) {
        const int round = grid.units / p.KVH, k = item / round;   // items of a head in a round
        if (round * p.KVH == grid.units && (k & 1)) item = k * round + min(round, total - k * round) - 1 - (item - k * round);
    }
    int early = 0;   // blocks in front of the pieces (pieces are between half and all of `most`)
    if (cut.total > 0 && sequences.per_lane == 1) {
        const Sequence& q = sequences.own;
        early = read_lane(wave_scan(max(uncut_of(q) - first_of(q, most * 3 / 4 + 1), 0)), kWaveSize - 1);
    }
    const int at = item - early;   // of the pieces
    const bool is_piece = at >= 0 && at < cut.total;
    int j, piece = 0;
    Sequence seq;
    if (is_piece) {
        int x = at;
        o.b = wave_uniform(cut.find(x));
        seq = sequences.at(o.b);
        const int per_block = pieces_of(tiles_of(seq.kv)), behind = int(unsigned(x) / unsigned(per_block));
        j = seq.blocks - 1 - behind;
        piece = x - behind * per_block;
    } else if (sequences.per_lane == 1) {
        // the (item - cut.total)th longest: the largest t so that more blocks than that have at least t tiles
        const int rank = at < 0 ? item : item - cut.total;
        const Sequence& q = sequences.own;
        const int end = uncut_of(q);
        int t = 0, behind = 0;   // behind: blocks of more than t tiles
        for (int hi = min(longest, most) + 1; hi - t > 1;) {
            const int mid = (t + hi) >> 1;
            const int count = read_lane(wave_scan(max(end - first_of(q, mid), 0)), kWaveSize - 1);
            if (count > rank) {
                t = mid;
            } else {
                hi = mid;
                behind = count;
            }
        }
        const int from = t == 0 ? 0 : min(first_of(q, t), end), to = min(first_of(q, t + 1), end);
        const int upto = wave_scan(to - from);
        int x = rank - behind;
        o.b = min(__builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x) | uint64_t(1) << 63), p.step.seqs - 1);
        if (o.b > 0) x -= read_lane(upto, o.b - 1);
        seq = sequences.at(o.b);
        j = read_lane(from, o.b) + x;
    } else {   // more sequences than lanes: not in order of their length, but the longest of each first (64 sequences, us in order
               // and, with an empty one more, out of it: prompts of 30 to 700 tokens 61, 66; of 30 to 2000 194, 199, at head size
               // 128 387, 396; three prompts' pieces beside 61 single rows 78, 88, at 128 116, 160)
        int x = item - cut.total;
        o.b = wave_uniform(whole.find(x));
        seq = sequences.at(o.b);
        j = uncut_of(seq) - 1 - x;
    }
    const int tokens = seq.tokens(j, positions), tiles = tiles_of(tokens), count = is_piece ? pieces_of(tiles) : 1;
    o.row = seq.row + j * positions;
    o.first = seq.kv - seq.n + j * positions;
    o.kv = seq.kv;
    o.slot = is_piece ? o.kvh * cut.total + at : -1;
    const int rows = min(seq.n - j * positions, positions);
    if (o.slot >= 0) {
        CutBlock& entry = grid.cuts[1 + o.slot];
        entry.row = o.row; entry.rows = rows; entry.kvh = o.kvh;
        entry.first = o.slot; entry.next = o.slot + 1; entry.stride = 1;
        entry.pieces = piece == 0 ? count : 0;
    }
    if (piece >= count || j < 0 || rows <= 0) return o;
    o.rows = rows;
    o.t_first = 0;
    o.t_stop = tokens;
    if (count > 1) {
        o.t_first = int(quotient(int64_t(tiles) * piece, count)) * kTile;
        o.t_stop = min(int(quotient(int64_t(tiles) * (piece + 1), count)) * kTile, tokens);
    }
    return o;
}

// Wide blocks.  Bound by the matrix pipe at head size 128 (2048 rows behind 14336 tokens, 32/8 heads: 460 us, 1.12 PFLOP/s, 478 on
// another device; a large matrix product reaches 1.23) and by the vector instructions of the softmax beside it at 64, where a tile's 32 exponentials
// a lane, at a quarter of the vector rate, take nearly as long as its 36 matrix instructions (4096 rows behind 4096 tokens: 249
// us, 0.83 PFLOP/s).  Short calls are their start: workgroups begin over 4 us, find their item, and have their first tile 2.4 us later
// (eight prompts of 134 to 1120 tokens: 29 us, of which the tiles are 11).  Four or two workgroups share a compute unit, so
// that one's softmax runs beside the other's matrix instructions.
template <int HD, int WPE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
attn_paged_wide_kernel(const PagedAttnParams p, const PagedGrid grid) {
    __shared__ __align__(1024) unsigned char s_stage0[WideTile<HD>::STAGE];   // (two arrays, so that the compiler can tell reads of one
    __shared__ __align__(1024) unsigned char s_stage1[WideTile<HD>::STAGE];   // from loads into the other)
    __shared__ OddValues<HD> odd;
    __shared__ WideItem s_item;
    const int rows_end = p.step.q_offsets[p.step.seqs], rows_begin = p.step.q_offsets[0];
    odd.clear();
    if (wave_uniform(int(threadIdx.x) / kWaveSize) == 0) {
        const WideItem item = wide_item<HD, WPE>(p, grid);
        if (threadIdx.x == 0) s_item = item;
    }
    __syncthreads();
    if (s_item.rows < 0) {
        clear_other_rows<HD>(p, p.step.rows, p.step.rows);
        return;
    }
    clear_other_rows<HD>(p, rows_begin, rows_end);
    if (s_item.rows == 0) return;
    WideItem o = s_item;
    o.b = wave_uniform(o.b); o.kvh = wave_uniform(o.kvh); o.kv = wave_uniform(o.kv);
    o.row = wave_uniform(o.row); o.rows = wave_uniform(o.rows); o.first = wave_uniform(o.first);
    o.t_first = wave_uniform(o.t_first); o.t_stop = wave_uniform(o.t_stop); o.slot = wave_uniform(o.slot);
    const PagedHead head = head_of(p, o.kv, o.b, o.kvh);
    char* const slot = o.slot >= 0 ? grid.slots + int64_t(o.slot) * wide_slot_bytes(HD, 2) : nullptr;
    if (wave_uniform(o.two)) wide_block<HD, 2, WPE>(p, head, o.kvh, o.row, o.rows, o.first, o.t_first, o.t_stop, slot, grid.units, s_stage0, s_stage1, odd);
    else wide_block<HD, 1, WPE>(p, head, o.kvh, o.row, o.rows, o.first, o.t_first, o.t_stop, slot, grid.units, s_stage0, s_stage1, odd);
}

// Narrow blocks of CB times 16 columns.  Bound by the bytes of keys and values: 64 sequences of 100 to 8191 tokens, 8 kv heads of
// 128, 477 MB in 80 us (6.0 TB/s; a pure read reaches 6.7), three of 60000 to 131071 tokens 1.07 GB in 166 us (6.4).  Every
// tile's loads are in flight while the one before is multiplied; two workgroups to a compute unit keep some 64 KiB on their way.
// One part a workgroup, all of one weight: none ends long before the others.  What is not tiles is 3 us of search in front and
// the last launch, 4 to 6 us (24 sequences with 2 to 7 drafted rows: 160 MB, 38 + 6 us).
template <int HD, int LOADS, int CB, int WPE>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
attn_paged_narrow_kernel(const PagedAttnParams p, const PagedGrid grid) {
    __shared__ __align__(1024) unsigned char s_mem[kWaves * NarrowArea<HD, LOADS, CB>::BYTES];
    __shared__ OddValues<HD> odd;
    const int tid = threadIdx.x, id = blockIdx.x, positions = CB * p.positions;
    const PagedStep& s = p.step;
    const Sequences sequences(p, CB);
    const int rows_end = s.q_offsets[s.seqs], rows_begin = s.q_offsets[0];
    odd.clear();
    __syncthreads();

    // How many parts: one per workgroup, fewer where there is little to do.  A part weighs at least kLeastChunk, so that the
    // places where consecutive parts cut a block are different tiles; where nothing is cut what a block of 16 tokens does, so
    // that none but the shortest share a part as long as there are enough (one sequence of 30 tokens 8.0 us otherwise, 5.4).  Whole eights, where there are as many, and consecutive
    // parts on one XCD: what a kv head's blocks share then stays in its cache.
    // Only sequences that do not overlap keep the weights within 64 bits: where offsets decrease the line is empty.
    bool falls = false;
    auto weight_of = [&](const Sequence& q) {
        falls |= q.falls;
        return q.weight(q.blocks, positions);
    };
    const Shares<int64_t, decltype(weight_of)> line(sequences, weight_of);
    if (__builtin_amdgcn_ballot_w64(falls) != 0) {
        if (grid.slots && tid == 0 && id == 0) grid.cuts[0].pieces = 0;
        clear_other_rows<HD>(p, s.rows, s.rows);
        return;
    }
    const int64_t total = line.total * p.KVH;
    int parts = int(std::max<int64_t>(1, std::min<int64_t>(gridDim.x, total / (grid.slots ? kLeastChunk : kBlockWeight + 16))));
    if (parts >= kXcds) parts &= ~(kXcds - 1);
    const int mine = id < parts && parts >= kXcds ? (id % kXcds) * (parts / kXcds) + id / kXcds : id;
    if (grid.slots && tid == 0) {
        grid.cuts[1 + mine].pieces = grid.cuts[1 + mine].ends = 0;
        if (id == 0) grid.cuts[0].pieces = parts;
    }

    clear_other_rows<HD>(p, rows_begin, rows_end);
    if (total == 0 || id >= parts) return;

    const int64_t per_part = quotient(total, parts);
    const int larger = int(total - per_part * parts);   // parts that weigh one more
    auto part_begin = [&](int part) { return per_part * part + min(part, larger); };
    const int64_t at = part_begin(mine), end = part_begin(mine + 1);
    int kvh = int(quotient(at, line.total));
    int64_t x = at - kvh * line.total;    // place in the head's line, then in the sequence
    int b = wave_uniform(line.find(x));
    Sequence seq = sequences.at(b);
    int j = 0;
    for (int span = seq.blocks; span > 1;) {   // the block that holds x: the last whose beginning is not behind it
        const int half = span / 2;
        if (seq.weight(j + half, positions) <= x) {
            j += half;
            span -= half;
        } else {
            span = half;
        }
    }
    int64_t begin = at - (x - seq.weight(j, positions));  // the block's place in the whole line
    while (true) {
        const int tokens = seq.tokens(j, positions);
        const int64_t weight = int64_t(seq.past()) + int64_t(j + 1) * positions + kBlockWeight;
        // where the block may be cut: whole tiles, and no slivers
        auto cut = [&](int64_t place) -> int {
            if (place <= 0 || !grid.slots) return 0;
            const int64_t t = ((place + kTile / 2) >> 6) << 6;
            static_assert(kTile == 64, "");
            return t < kLeastPiece ? 0 : t > tokens - kLeastPiece ? tokens : int(t);
        };
        const int t_first = cut(at - begin);
        const int t_stop = (end - begin >= weight) ? tokens : cut(end - begin);
        const bool whole = t_first == 0 && t_stop == tokens;
        if (t_first < t_stop || (tokens == 0 && at <= begin)) {
            const int row = seq.row + j * positions, rows = min(seq.n - j * positions, positions);
            if (!whole && tid == 0) {
                CutBlock& entry = grid.cuts[1 + mine];
                if (t_first == 0) {
                    entry.row = row; entry.rows = rows; entry.kvh = kvh;
                    entry.first = 2 * mine + 1; entry.next = 2 * (mine + 1); entry.stride = 2;   // (two slots a part: a block that it ends, one that it begins)
                    entry.pieces = 1;
                } else {
                    entry.ends = t_stop == tokens;
                }
            }
            narrow_block<HD, LOADS, CB>(p, head_of(p, seq.kv, b, kvh), kvh, row, rows, seq.kv - seq.n + j * positions, t_first, t_stop,
                                        whole ? nullptr : grid.slots + int64_t(2 * mine + (t_first == 0)) * narrow_slot_bytes(HD, CB), s_mem, odd);
        }

        begin += weight;
        if (begin >= end) break;
        ++j;
        while (j >= seq.blocks) {   // the next sequence with narrow blocks, or the next head's first (there is one: the line goes on)
            j = 0;
            if (++b == s.seqs) {
                b = 0;
                if (++kvh >= p.KVH) return;   // (the line's end is the last head's: begin has reached `end`)
            }
            seq = sequences.at(b);
        }
    }
}

// What a thread adds up of a block that was cut: n groups of four dims, 16 apart, of one row and head.
template <int HD, int N>
__device__ __forceinline__ void merge_pieces(const PagedAttnParams& p, const CutBlock& block, const char* slots, int64_t slot_bytes, int row, int h, int dim,
                                             int at, int step, int at_ml) {
    constexpr int G = N == 1 ? 16 : 4;   // pieces whose reads are in flight together
    f32x4_t sum[N];
    float total = 0.f, M = kNothing;
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < block.pieces; i0 += G) {
        f32x4_t o[G][N];
        float2 ml[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int piece = min(i0 + g, block.pieces - 1);
            const char* const from = slots + (piece == 0 ? block.first : block.next + (piece - 1) * block.stride) * slot_bytes;
            ml[g] = *reinterpret_cast<const float2*>(from + at_ml);
#pragma unroll
            for (int i = 0; i < N; ++i) o[g][i] = *reinterpret_cast<const f32x4_t*>(from + at + i * step);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (i0 + g < block.pieces) {
                const float m_new = fmaxf(M, ml[g].x);
                const float old = fast_exp2((M - m_new) * p.scale_log2e), f = fast_exp2((ml[g].x - m_new) * p.scale_log2e);
                M = m_new;
                total = fmaf(ml[g].y, f, total * old);
#pragma unroll
                for (int i = 0; i < N; ++i) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[i][r] = fmaf(o[g][i][r], f, sum[i][r] * old);
                }
            }
        }
    }
    // A block that was cut has more tokens than rows and its last row sees them all, so every row sees some: the sum is 0 only
    // where all their scores are minus infinity, and the row NaN then, as in a block that was not cut.
    static_assert(kLeastWidePiece * kTile > 8 * 16 && 2 * kLeastPiece > 2 * 16, "tokens of a block that is cut; rows of a block");
    const float inv = 1.0f / total;
    uint16_t* const out = p.out + int64_t(row) * p.o_sr + h * p.o_sh + dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        *reinterpret_cast<uint2*>(out + i * 16) = make_uint2(pack_bf16x2(sum[i][0] * inv, sum[i][1] * inv), pack_bf16x2(sum[i][2] * inv, sum[i][3] * inv));
    }
}

// Adds up the pieces of the blocks that were cut, in their order: partial results written and read once, 4 to 6 us behind narrow
// blocks (4 of them a launch that finds nothing), 10 behind 900 pieces of wide ones (33 MB).  Workgroup (c, y): the block of entry c, the y-th group of
// its dims.
template <int HD, int NARROW>
__global__ void __launch_bounds__(kThreads) attn_paged_merge_kernel(const PagedAttnParams p, const PagedGrid grid, const int bits) {
    constexpr int NB = HD / 16, WIDE = 2;   // (only blocks of two column blocks are cut)
    const int tid = threadIdx.x, y = blockIdx.y, entries = grid.cuts[0].pieces;
    // The blocks that were cut are some of the entries, often ones a power of two apart.  Workgroups take them in the order
    // of their reversed bits, so that those do not all run on one XCD (128 blocks of 8 pieces: 33 us on one).
    for (int c = blockIdx.x; c < 1 << bits; c += int(gridDim.x)) {
        const int e = int(__builtin_bitreverse32(unsigned(c)) >> (32 - bits));
        if (e >= entries) continue;
        CutBlock block = grid.cuts[1 + e];
        if (block.pieces == 0) continue;
        if constexpr (NARROW > 0) {
            // its pieces: up to the next part that ends a block
            for (int from = e + 1; from < entries; from += kWaveSize) {
                const int part = from + (tid & (kWaveSize - 1));
                const uint64_t here = __builtin_amdgcn_ballot_w64(part < entries && grid.cuts[1 + part].ends != 0);
                if (here) {
                    block.pieces = from + __builtin_ctzll(here) - e + 1;
                    break;
                }
            }
            const int item = y * kThreads + tid, column = item / (HD / 4), dim = item % (HD / 4) * 4;
            const int fn = column % 16, of = fn * p.inverse >> 8, i = column / 16 * p.positions + of;
            if (of >= p.positions || i >= block.rows) continue;
            merge_pieces<HD, 1>(p, block, grid.slots, narrow_slot_bytes(HD, NARROW), block.row + i, block.kvh * p.R + fn - of * p.R, dim,
                                (column * HD + dim) * 4, 0, NARROW * 16 * HD * 4 + column * 8);
        } else {
            const int lane = tid & (kWaveSize - 1), wave = tid / kWaveSize, fn = lane & 15, fg = lane >> 4;
            const int cb = y / (NB / 4), nb0 = y % (NB / 4) * 4;
            const int of = fn * p.inverse >> 8, i = (wave * WIDE + cb) * p.positions + of;
            if (of >= p.positions || i >= block.rows) continue;
            merge_pieces<HD, 4>(p, block, grid.slots, wide_slot_bytes(HD, WIDE), block.row + i, block.kvh * p.R + fn - of * p.R, nb0 * 16 + fg * 4,
                                ((cb * NB + nb0) * kThreads + tid) * 16, kThreads * 16, WIDE * NB * kThreads * 16 + (cb * kThreads + tid) * 8);
        }
    }
}

// Workgroups that share a compute unit (wavefronts per SIMD).
constexpr int wide_wpe(int HD) { return HD == 64 ? 4 : 2; }
constexpr int kNarrowWpe = 2;

// Sizes of a call's launches, from what the host knows.
struct Sizes {
    int narrow;   // column blocks of the narrow form; 0: the wide form
    int64_t workgroups;
    int entries;
    size_t slots, cuts;   // bytes
};
Sizes sizes_of(const PagedStep& s, int QH, int KVH, int HD, int max_new) {
    const int R = QH / KVH, ppb = 16 / R, cus = current_device_cus();
    const int64_t rows = max_new > 0 ? std::min(max_new, s.rows) : s.rows;   // of a sequence at most
    Sizes z = {};
    // Narrow up to two column blocks (more would be two streams of the same tokens).  us of the narrow and of the wide form, rows to
    // a sequence on either side of the line: head size 128, four heads to a kv head, 24 sequences of 500 to 4001 tokens: 4 rows 46, 51;
    // 8 rows 50, 53; 9 rows 75, 56; 16 rows 81, 59; 4 sequences of 1500: 8 rows 21, 30; 9 rows 22, 31; 16 rows 24, 31.  Head size 64: 8 rows 31,
    // 26; 9 rows 41, 28; of 4 sequences 15, 22; 15, 21.  Sixteen heads to a kv head, 128: 2 rows 33, 27; 3 rows 44, 31; of 4 sequences 19,
    // 30; 19, 31.  One head, 128: 32 rows 50, 52; 33 rows 76, 55; of 4 sequences 21, 30; 23, 31.  (Few sequences would have the narrow form a
    // little further: how many there are is known, how long they are is not.)
    if (rows <= 2 * ppb) {
        z.narrow = rows > ppb ? 2 : 1;
        z.workgroups = z.entries = kNarrowWpe * cus / kXcds * kXcds;
        // few tokens: what a cut saves is less than the last launch costs (by the table: one of 30 tokens has it at 8192, 9.6 us for 5.2)
        if (s.max_kv <= kLeastCut) z.entries = 0;
        z.slots = size_t(z.entries) * 2 * narrow_slot_bytes(HD, z.narrow);
    } else {
        // blocks: every sequence may end with one that is not full.  Pieces: at most four to a compute unit; where the
        // blocks alone keep the device busy none is cut, however long one of them (head size 128, 8 kv heads, a piece of 300 rows
        // beside one row behind 131071 tokens and 200 of 500: 213 us; 260 of them are that many blocks: 2.3 ms).
        auto blocks_of = [&](int cb) { return (s.rows / (ppb * kWaves * cb) + std::min(s.seqs, s.rows)) * int64_t(KVH); };
        const int residents = wide_wpe(HD) * cus;
        if (blocks_of(2) < 4 * residents && s.max_kv > kLeastWideCut) z.entries = 4 * cus;
        z.workgroups = blocks_of(1) + z.entries;
        z.slots = size_t(z.entries) * wide_slot_bytes(HD, 2);
    }
    if (z.entries > 0) z.cuts = (size_t(z.entries) + 1) * sizeof(CutBlock);
    return z;
}

template <int HD, int NARROW>
int launch(const PagedAttnParams& p, const Sizes& z, void* workspace, hipStream_t stream) {
    char* const memory = static_cast<char*>(workspace);
    const PagedGrid grid = {memory, reinterpret_cast<CutBlock*>(memory ? memory + z.slots : nullptr), memory ? z.entries : 0, current_device_cus()};
    const dim3 workgroups(unsigned(z.workgroups)), threads(kThreads);
    int rc;
    if constexpr (NARROW > 0) rc = enqueue(attn_paged_narrow_kernel<HD, 8, NARROW, kNarrowWpe>, workgroups, threads, 0, stream, p, grid);
    else rc = enqueue(attn_paged_wide_kernel<HD, wide_wpe(HD)>, workgroups, threads, 0, stream, p, grid);
    if (rc != 0 || grid.entries == 0) return rc;
    const int groups = NARROW > 0 ? NARROW * 16 * HD / 4 / kThreads : 2 * HD / 64;
    int bits = 1;
    while (1 << bits < z.entries) ++bits;
    const int merging = std::min(z.entries, 2 * current_device_cus());
    return enqueue(attn_paged_merge_kernel<HD, NARROW>, dim3(unsigned(merging), unsigned(groups)), threads, 0, stream, p, grid, bits);
}

template <int HD>
int launch_of(const PagedAttnParams& p, const Sizes& z, void* workspace, hipStream_t stream) {
    if (z.narrow > 0) return z.narrow == 1 ? launch<HD, 1>(p, z, workspace, stream) : launch<HD, 2>(p, z, workspace, stream);
    return launch<HD, 0>(p, z, workspace, stream);
}

}  // namespace

bool attn_paged_fits(const PagedStep& step, int QH, int KVH, int HD, int max_new) {
    return sizes_of(step, QH, KVH, HD, max_new).workgroups * kThreads < int64_t(1) << 32;
}

size_t attn_paged_workspace_bytes(const PagedStep& step, int QH, int KVH, int HD, int max_new) {
    const Sizes z = sizes_of(step, QH, KVH, HD, max_new);
    return z.slots + z.cuts;
}

int launch_attn_paged(const PagedAttnParams& p, int HD, void* workspace, hipStream_t stream) {
    const Sizes z = sizes_of(p.step, p.QH, p.KVH, HD, p.max_new);
    return HD == 64 ? launch_of<64>(p, z, workspace, stream) : launch_of<128>(p, z, workspace, stream);
}

}  // namespace l3
