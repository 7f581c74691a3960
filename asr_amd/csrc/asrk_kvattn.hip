// Attention over the paged 8-bit cache:  o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(c q.k_t - m),  c = scale log2(e),  in one
// pass over the tokens with a running maximum m.
//
// HBM-bound for single tokens (2 D bytes per token and head against 4 D G flops), so the kernel is built around the page:
// a wave takes whole pages of 64 tokens straight from memory into registers with 16-byte loads, no LDS and no shuffle
// between the two products.  What makes that work is that a product may run over its inner index in any order, as long as
// both operands use the same one:
//   S^T = K Q^T   (16x16x32 bf16)  rows of tile t are tokens 16 (r >> 2) + 4 t + (r & 3), so that lane (column c, group g)
//                                  ends up with tokens 16 g .. 16 g + 15 of column c over the four tiles;
//                                  the inner index is read 16 d's per lane at a time, and q is laid out the same way
//   O^T = V^T P^T (16x16x32 f16)   the lane's 16 weights are the second operand as they are, and 16 consecutive tokens of
//                                  one d are 16 bytes of the value page
// Columns are the rows of q that share a key/value head: beams x new tokens x query heads per key/value head.
// Keys become bf16 with their scale applied (exact); values become f16 in a unit that follows the pages' scales (exact, see
// Unit).  Weights are rounded to f16, 2^-11 relative, 8 times finer than bf16 would be and well under the 2^-8 of the bf16
// result.  Everything else is fp32.
// Measured: 1.2 GB of cache (48 sequences, 8 heads of 128) 203 us = 5.9 TB/s; 64 x 5 beams over 1641 tokens that share their
// prompts (64 MB) 20 us; one utterance 11 us, latency, of which fetching the code for the first time is a good part.
#include "asrk_kvcache.h"

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

constexpr int NO_COLUMN = 0x7fffffff;  // limit of a lane behind the last column: takes part in nothing, and masks nothing
constexpr float NEG_INF = -__builtin_inff();

// In a block that a uniform condition rarely enters: without it the compiler computes both sides and selects, which costs
// the common path more vector instructions than its own work.
#define KEEP_BRANCH() asm volatile("")

struct AttnArgs {
    const bf16_t* q;
    bf16_t* out;
    float* part_o;   // [splits][S n Hq][D]
    float2* part_ml; // [splits][S n Hq]
    int64_t seq_ld, row_ld, head_ld, layer, rows;  // rows: S n Hq
    double per_seq_inv, group_inv;  // 1 / (n group), 1 / group: a division by a runtime integer is 30 instructions
    int n, group, beams, splits;    // new tokens, query heads per key/value head
    float c;
};

__device__ __forceinline__ float pow2(int e) {  // any e; below the normal range: 0
    return e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23);
}

template <bool HI>
__device__ __forceinline__ bf16x2 k2(uint32_t w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI); }
template <bool HI>
__device__ __forceinline__ f16x2 v2(uint32_t w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, HI); }
__device__ __forceinline__ bf16x8 k8(uint32_t a, uint32_t b, float s) {
    const bf16x2 r0 = k2<false>(a, s), r1 = k2<true>(a, s), r2 = k2<false>(b, s), r3 = k2<true>(b, s);
    return bf16x8{r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}
__device__ __forceinline__ f16x8 v8(uint32_t a, uint32_t b, float s) {
    const f16x2 r0 = v2<false>(a, s), r1 = v2<true>(a, s), r2 = v2<false>(b, s), r3 = v2<true>(b, s);
    return f16x8{r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}

// 0xff in every byte of w that is an e4m3 NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    const uint32_t is = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return (is >> 7) * 0xffu;
}

// Maximum over the lanes of a column's four groups, and over all lanes of a wave.
__device__ __forceinline__ float groups_max(float v) {  // rows of 16 lanes, then halves, exchanged in registers
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ int over(int x, double inverse) { return (int)(((double)x + 0.5) * inverse); }  // exact

// Grid: x: (head, split), y: set of sequences, z: chunk of columns; whole waves in this order.
__device__ __forceinline__ int head_of(const AttnArgs& a) { return a.splits == 1 ? blockIdx.x : blockIdx.x / (unsigned)a.splits; }
__device__ __forceinline__ int part_of(const AttnArgs& a) { return a.splits == 1 ? 0 : blockIdx.x % (unsigned)a.splits; }

// Column y of a set of sequences: beam, new token, query head.
struct Columns {
    const AttnArgs& a;
    int set, h, H, per_seq, columns;
    __device__ __forceinline__ Columns(const asrk_kv_cache& c, const AttnArgs& args, int set_)
        : a(args), set(set_), h(head_of(args)), H(c.kv_heads), per_seq(args.n * args.group), columns(args.beams * per_seq) {}
    __device__ __forceinline__ void split(int y, int& b, int& i, int& j) const {
        b = over(y, a.per_seq_inv);
        const int in = y - b * per_seq;
        i = over(in, a.group_inv);
        j = in - i * a.group;
    }
    __device__ __forceinline__ int64_t row_of(int y) const {  // of out, in units of D
        int b, i, j;
        split(y, b, i, j);
        return (((int64_t)set * a.beams + b) * a.n + i) * (int64_t)(H * a.group) + h * a.group + j;
    }
};

// What a lane holds of its CT columns: q as the second operand (16 consecutive d's per pair of steps), the beam, the number
// of tokens seen; the largest such number of the lane.
template <int D, int CT>
struct Queries {
    bf16x8 q[CT][D / 32];
    int limit[CT], beam[CT], most;
    __device__ __forceinline__ void load(const asrk_kv_cache& c, const Columns& cs, int first_col, int col, int g) {
        const int top = c.max_pages * ASRK_KV_PAGE;
        most = 0;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int x = first_col + 16 * t + col;
            beam[t] = 0;
            limit[t] = NO_COLUMN;
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) q[t][s][e] = (bf16_t)0.f;
            if (x < cs.columns) {
                int b, i, j;
                cs.split(x, b, i, j);
                const int64_t seq = (int64_t)cs.set * cs.a.beams + b;
                const int start = c.starts[seq * c.seq_stride], fresh = c.lens[seq * c.seq_stride] - start;
                beam[t] = b;
                limit[t] = i >= fresh ? 0 : (start + i + 1 < top ? start + i + 1 : top);
                most = limit[t] > most ? limit[t] : most;
                const bf16_t* p = cs.a.q + seq * cs.a.seq_ld + (int64_t)i * cs.a.row_ld + (int64_t)(cs.h * cs.a.group + j) * cs.a.head_ld + 16 * g;
#pragma unroll
                for (int s = 0; s < D / 64; ++s) {
                    q[t][2 * s] = *reinterpret_cast<const bf16x8*>(p + 64 * s);
                    q[t][2 * s + 1] = *reinterpret_cast<const bf16x8*>(p + 64 * s + 8);
                }
            }
        }
    }
    // Of page p, for the beams `with`: tokens seen by each column; whether all see all of it, and whether any sees any.
    __device__ __forceinline__ bool see(int p, uint64_t with, int* seen, bool& whole) const {
        int all = ASRK_KV_PAGE, some = 0;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const int s = limit[t] - p * ASRK_KV_PAGE;
            const bool takes = ((uint32_t)with >> beam[t]) & 1;  // 32 beams at most: one register
            seen[t] = limit[t] == NO_COLUMN || (takes && s > ASRK_KV_PAGE) ? ASRK_KV_PAGE : (takes && s > 0 ? s : 0);
            all = seen[t] < all ? seen[t] : all;
            some = seen[t] > some && limit[t] != NO_COLUMN ? seen[t] : some;
        }
        whole = __all(all == ASRK_KV_PAGE);
        return __any(some > 0);
    }
};

// The work on a set of sequences, page by page: beams whose tables agree on a page take it together.
struct Item {
    int page, p;  // -1: no more; the p-th page of its sequences
    uint64_t with;
};
struct Pages {
    const int* table;  // of beam `lane`
    int beams, max_pages, num_pages, lane, at_p, step, item_p, mine, coming;
    uint64_t left;
    __device__ __forceinline__ Pages(const asrk_kv_cache& c, int beams_, int set, int first, int step_, int lane_)
        : beams(beams_), max_pages(c.max_pages), num_pages(c.num_pages), lane(lane_), at_p(first), step(step_), item_p(0),
          mine(-1), left(0) {
        table = c.table + ((int64_t)set * beams + lane) * c.seq_stride * max_pages;
        coming = number(first);
    }
    __device__ __forceinline__ int number(int p) const { return lane < beams && p < max_pages ? table[p] : -1; }
    __device__ __forceinline__ Item next(int pages) {
        while (!left) {
            if (at_p >= pages) return Item{-1, 0, 0};
            mine = coming;
            item_p = at_p;
            at_p += step;
            coming = number(at_p);  // on its way a page ahead
            left = __ballot(mine >= 0 && mine < num_pages);
        }
        const int page = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t with = __ballot(mine == page) & left;
        left &= ~with;
        return Item{page, item_p, with};
    }
};

// Loads go through a descriptor of the page: one register of lane offset, the rest in the instruction.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const char* layer, int64_t at, int D) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform_ptr(layer + at * (2 * ASRK_KV_PAGE * D))), 0, 2 * ASRK_KV_PAGE * D,
                                             0x00020000);
}

// Bytes of the lane's 16 tokens that lie before token `last` of the page (behind the last token the page may hold anything).
__device__ __forceinline__ u32x4 keep_before(int last, int g) {
    u32x4 mask;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int keep = last - 16 * g - 4 * w;
        mask[w] = (uint32_t)((1ull << (8 * (keep < 0 ? 0 : (keep > 4 ? 4 : keep)))) - 1);
    }
    return mask;
}
// Values are multiplied, and o is held, in units of 2^now.  An e4m3 value times 2^-15 .. 2^7 is exact in f16, so the unit
// stays while a page's exponent lies in that window, and else follows it up or down.  (A unit that only rises would round the
// values of a beam, or of a page, by those of another that happens to come before.)  That does while all exponents so far lie
// within 2^64: o, at most 2^(64 + 7) times what a page adds to it (2^24 per token at most), cannot leave fp32's range then.
// Exponents further apart -- of beams that are worked on together, or of pages whose weights make up for it or not -- leave no
// unit in which f16 holds both: walk_apart() takes over.
struct Unit {
    int now = ASRK_KV_EXP_MIN, low = ASRK_KV_EXP_MAX, high = ASRK_KV_EXP_MIN;
    __device__ __forceinline__ bool follow(int ev) {  // false: too far apart
        low = ev < low ? ev : low;
        high = ev > high ? ev : high;
        const int d = ev - now;
        if (d > 7 || d < -15) now = ev;
        return high - low <= 64;
    }
};

// Scores of one page to weights, 2^HEAD times what they are to the reference: f16's range is spent on the small ones.  A
// weight of 2^-27 of the largest still has all 11 bits, and below that it is held to 2^-38 of the largest.  The reference
// follows the maximum only when that has grown by more than 2^SLACK: up to there nothing overflows (2^15) and o and the sum
// need no rescaling.
// Where scores pass 2^20 or so, their neighbouring fp32 numbers lie far apart and the reference is off by that much; so it is
// rounded down, and a weight cut at f16's largest number: scores closer than two of those neighbours then count the same (the cut
// costs 2 % of the prompts' time; branches for such scores would cost single tokens 10 %).
constexpr float HEAD = 13.f, SLACK = 2.f;
template <int CT, int DT>
__device__ __forceinline__ void weigh(f32x4 (*sc)[4], const int* seen, bool whole, int g, float scale, int up, int unit, float* m, f32x4* l,
                                      f32x4 (*o)[DT], f16x8 (*pf)[2]) {
    const float shrink = pow2(unit - up);
    constexpr _Float16 MOST = 65504.f;
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        if (!whole) {
            KEEP_BRANCH();
            const int mine = seen[x] - 16 * g;  // of the lane's 16 tokens
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[x][t][i] = 4 * t + i < mine ? sc[x][t][i] : NEG_INF;
        }
        float top = NEG_INF;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[x][t][i]);
        const float now = groups_max(top) * scale;  // scale > 0
        if (__any(now > m[x] + SLACK) || up != unit) {
            KEEP_BRANCH();
            const float low = fmaf(fabsf(now), -0x1p-23f, now);  // +inf: NaN, as the result has to be
            const float to = now > m[x] + SLACK && !(low <= m[x]) ? low : m[x];  // by the column alone: its bits do not depend on its neighbours
            const float back = to > NEG_INF ? __builtin_amdgcn_exp2f(m[x] - to) : 0.f;
            m[x] = to;
#pragma unroll
            for (int i = 0; i < 4; ++i) l[x][i] *= back;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[x][d] *= back * shrink;
        }
        const float ref = m[x] == NEG_INF ? 0.f : m[x] - HEAD;  // nothing seen yet: every weight is 0
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const f32x2_t w = {__builtin_amdgcn_exp2f(fmaf(sc[x][t][i], scale, -ref)),
                                   __builtin_amdgcn_exp2f(fmaf(sc[x][t][i + 1], scale, -ref))};
                const f16x2 h = __builtin_elementwise_minimum(__builtin_convertvector(w, f16x2), f16x2{MOST, MOST});  // to nearest; NaN stays
                pf[x][t >> 1][4 * (t & 1) + i] = h[0];
                pf[x][t >> 1][4 * (t & 1) + i + 1] = h[1];
            }
    }
}

// The sum of the weights as they are used: a product with ones, all four rows of a lane are the column's sum.
template <int CT>
__device__ __forceinline__ void add_weights(const f16x8 (*pf)[2], f32x4* l) {
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int x = 0; x < CT; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) l[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[x][u], l[x], 0, 0, 0);
}

// A page whose values hold a NaN (rare: the page says so).  0 * NaN must not reach columns that do not see its token, so the
// NaNs were made zeros for the product; here what a product of the 0/1 patterns (is a NaN, is seen) says becomes NaN.
template <int CT, int DT, class Load>
__device__ __forceinline__ void mark_nans(Load&& raw_value, const int* seen, int g, f32x4 (*o)[DT]) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        __builtin_amdgcn_sched_barrier(0);  // one tile at a time: this path must not cost the other one registers
        const u32x4 raw = raw_value(d);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
            f32x4 hit{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f16x8 sees;
#pragma unroll
                for (int i = 0; i < 8; ++i) sees[i] = 16 * g + 8 * u + i < seen[x] ? (_Float16)1.f : (_Float16)0.f;
                const f16x8 is = v8(nan_bytes(raw[2 * u]) & 0x38383838u, nan_bytes(raw[2 * u + 1]) & 0x38383838u, 1.f);  // 0x38 is 1
                hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees, hit, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[x][d][i] = hit[i] > 0.f ? __builtin_nanf("") : o[x][d][i];
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The pages from `item` on, where exponents lie further apart than one unit can hold: each is multiplied in the unit of its own
// exponent, from zero, and added to o in fp32, in units of 2^APART: all that a page can add lies in fp32's range (2^(119 + 9 +
// 15 - 44) per token at most).  Rare, so it must not cost the other loop registers: each wave reads and converts for itself, and
// takes one tile of anything at a time.
constexpr int APART = 44;
template <int D, int CT>
__device__ __forceinline__ void walk_apart(Item item, Pages& work, int pages, const Queries<D, CT>& qs, const Columns& cs, const char* layer,
                                           const int* exps, int lane, float* m, f32x4* l, f32x4 (*o)[D / 16]) {
    constexpr int KS = D / 64, DT = D / 16;
    const int col = lane & 15, g = lane >> 4;
    for (; item.page >= 0; item = work.next(pages)) {
        int seen[CT];
        bool whole;
        if (!qs.see(item.p, item.with, seen, whole)) continue;
        const int64_t at = (int64_t)item.page * cs.H + cs.h;
        const __amdgpu_buffer_rsrc_t rows = page_rows(layer, at, D);
        const int e = __builtin_amdgcn_readfirstlane(exps[at]);
        const float ks = pow2((int8_t)e), up = pow2((int8_t)(e >> 8) - APART);
        const bool odd = (e >> 16) & 1;
        int last = 0;  // token seen by any column
#pragma unroll
        for (int x = 0; x < CT; ++x) last = seen[x] > last && qs.limit[x] != NO_COLUMN ? seen[x] : last;
        const u32x4 mask = keep_before(wave_imax(last), g);
        auto value = [&](int d) __attribute__((always_inline)) {
            return __builtin_amdgcn_raw_buffer_load_b128(rows, (col + 16 * d) * ASRK_KV_PAGE + 16 * g, ASRK_KV_PAGE * D, 0);
        };
#pragma unroll
        for (int x = 0; x < CT; ++x) {  // one tile of columns, of keys, of values at a time
            f32x4 sc[1][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                sc[0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const u32x4 raw = __builtin_amdgcn_raw_buffer_load_b128(rows, (16 * (col >> 2) + 4 * t + (col & 3)) * D + 64 * s + 16 * g, 0, 0);
                    sc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8(raw[0], raw[1], ks), qs.q[x][2 * s], sc[0][t], 0, 0, 0);
                    sc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8(raw[2], raw[3], ks), qs.q[x][2 * s + 1], sc[0][t], 0, 0, 0);
                }
            }
            f16x8 pf[1][2];
            weigh<1, DT>(sc, seen + x, whole, g, cs.a.c, APART, APART, m + x, l + x, o + x, pf);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                __builtin_amdgcn_sched_barrier(0);
                u32x4 raw = value(d) & mask;
                if (odd)
#pragma unroll
                    for (int w = 0; w < 4; ++w) raw[w] &= ~nan_bytes(raw[w]);
                f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8(raw[2 * u], raw[2 * u + 1], 1.f), pf[0][u], sum, 0, 0, 0);
                o[x][d] += sum * up;
            }
            add_weights<1>(pf, l + x);
            if (odd) mark_nans<1, DT>(value, seen + x, g, o + x);
        }
    }
}

// The same from the first page on, with nothing of what the other loop holds: if it went on from there, that loop would be cut
// for both (two spilled registers more in kv_prompt_kernel<64>, 10 % of the time of 16 prompts).  Its presence still costs 1 to 4 %; a call
// that goes through it takes twice its time.
template <int D, int CT>
__device__ __forceinline__ void walk_apart_anew(const asrk_kv_cache& c, const Columns& cs, int first_col, int first_page, int step, int pages,
                                                const char* layer, const int* exps, float* m, f32x4* l, f32x4 (*o)[D / 16]) {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane));  // what follows from it is computed and loaded again
    Pages work(c, cs.a.beams, cs.set, first_page, step, lane);
    Queries<D, CT> qs;
    qs.load(c, cs, first_col, lane & 15, lane >> 4);
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        m[x] = NEG_INF;
        l[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    walk_apart<D, CT>(work.next(pages), work, pages, qs, cs, layer, exps, lane, m, l, o);
}

// f over groups of W lanes, in all of them.
template <int W, class F>
__device__ __forceinline__ float among(float v, F&& f) {
    auto lanes = [&](auto control) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), control.value, 0xf, 0xf, true)); };
    v = f(v, lanes(std::integral_constant<int, 0xB1>()));                   // 1 0 3 2
    v = f(v, lanes(std::integral_constant<int, 0x4E>()));                   // 2 3 0 1
    if (W == 8) v = f(v, lanes(std::integral_constant<int, 0x141>()));      // 7 6 5 4 3 2 1 0
    return v;
}

// Waves per SIMD that the registers are cut for: as many as hold a page, q, o and the scores without spilling in the loop.
// (D 64, 1 tile: 4; with 3, 64 x 5 beams take 24.5 us instead of 19.7.  D 128, 1 tile: 2; with 3 it spills and 1.2 GB of
// cache take 228 us instead of 204.)
constexpr int occupancy(int D, int CT) { return D == 64 ? (CT == 1 ? 4 : 3) : 2; }

// Few columns (single tokens): the W waves of a workgroup share CT tiles of 16 and deal the pages among them, and among
// the splits.  A wave takes a page straight into registers; the next page's keys are loaded over this one's as soon as the
// scores are done, its values as soon as they are used.
template <int D, int CT, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(occupancy(D, CT), occupancy(D, CT))))
void kv_attention_kernel(asrk_kv_cache c, AttnArgs a) {
    constexpr int KS = D / 64;   // 16-byte pieces of a key row per lane
    constexpr int DT = D / 16;   // tiles of 16 d
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int part = part_of(a), set = blockIdx.y;
    const Columns cs(c, a, set);
    const int first_col = blockIdx.z * 16 * CT;
    // The pages of a wave: by its number alone, so that their numbers are on the way before the lengths are known.
    Pages work(c, a.beams, set, part * W + wave, a.splits * W, lane);
    Queries<D, CT> qs;
    qs.load(c, cs, first_col, col, g);
    const int pages = (wave_imax(qs.most) + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE;

    f32x4 o[CT][DT], l[CT];
    float m[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        m[t] = NEG_INF;
        l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Unit unit;
    int held_unit = unit.now;  // of o

    const char* layer = (const char*)c.kv + a.layer * c.num_pages * cs.H * (int64_t)(2 * ASRK_KV_PAGE * D);
    const int* exps = (const int*)c.exps + a.layer * c.num_pages * cs.H;
    const uint32_t k_at = (16 * (col >> 2) + (col & 3)) * D + 16 * g, v_at = col * ASRK_KV_PAGE + 16 * g;  // this lane's bytes
    u32x4 kr[4][KS], vr[DT];
    auto load_keys = [&](__amdgpu_buffer_rsrc_t rows) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[t][s] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_at + 4 * t * D + 64 * s, 0, 0);
    };
    auto load_value = [&](__amdgpu_buffer_rsrc_t rows, int d) __attribute__((always_inline)) {
        return __builtin_amdgcn_raw_buffer_load_b128(rows, v_at + 16 * d * ASRK_KV_PAGE, ASRK_KV_PAGE * D, 0);
    };
    Item item = work.next(pages);
    int64_t at = (int64_t)(item.page < 0 ? 0 : item.page) * cs.H + cs.h;
    __amdgpu_buffer_rsrc_t rows = page_rows(layer, at, D);
    bool apart = false;
    if (item.page >= 0) {
        int e_next = exps[at];
        load_keys(rows);
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[d] = load_value(rows, d);
        for (;;) {
            const int e = __builtin_amdgcn_readfirstlane(e_next), ev = (int8_t)(e >> 8);
            if (__builtin_expect(!unit.follow(ev), 0)) {
                apart = true;
                break;
            }
            const int up = unit.now;
            const Item following = work.next(pages);
            at = (int64_t)(following.page < 0 ? 0 : following.page) * cs.H + cs.h;
            const __amdgpu_buffer_rsrc_t rows_next = page_rows(layer, at, D);
            if (following.page >= 0) e_next = exps[at];
            int seen[CT];
            bool whole;
            qs.see(item.p, item.with, seen, whole);

            const float ks = pow2((int8_t)e);
            f32x4 sc[CT][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int x = 0; x < CT; ++x) sc[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const bf16x8 k0 = k8(kr[t][s][0], kr[t][s][1], ks), k1 = k8(kr[t][s][2], kr[t][s][3], ks);
#pragma unroll
                    for (int x = 0; x < CT; ++x) {
                        sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qs.q[x][2 * s], sc[x][t], 0, 0, 0);
                        sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qs.q[x][2 * s + 1], sc[x][t], 0, 0, 0);
                    }
                }
            }
            if (following.page >= 0) load_keys(rows_next);
            f16x8 pf[CT][2];
            weigh<CT, DT>(sc, seen, whole, g, a.c, up, held_unit, m, l, o, pf);
            held_unit = up;
            const float vs = pow2(ev - up);
            if (!whole) {
                KEEP_BRANCH();
                int last = 0;  // token seen by any column
#pragma unroll
                for (int x = 0; x < CT; ++x) last = seen[x] > last && qs.limit[x] != NO_COLUMN ? seen[x] : last;
                const u32x4 mask = keep_before(wave_imax(last), g);
#pragma unroll
                for (int d = 0; d < DT; ++d) vr[d] &= mask;
            }
            const bool odd = __builtin_expect((e >> 16) & 1, 0);
            if (odd) {
                KEEP_BRANCH();
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int w = 0; w < 4; ++w) vr[d][w] &= ~nan_bytes(vr[d][w]);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const f16x8 v = v8(vr[d][2 * u], vr[d][2 * u + 1], vs);
#pragma unroll
                    for (int x = 0; x < CT; ++x) o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[x][u], o[x][d], 0, 0, 0);
                }
            add_weights<CT>(pf, l);
            if (odd) mark_nans<CT, DT>([&](int d) { return load_value(rows, d); }, seen, g, o);
            if (following.page >= 0) {
#pragma unroll
                for (int d = 0; d < DT; ++d) vr[d] = load_value(rows_next, d);
            }
            if (following.page < 0) break;
            item = following;
            rows = rows_next;
        }
    }
    if (__builtin_expect(apart, 0)) {
        held_unit = APART;
        walk_apart_anew<D, CT>(c, cs, first_col, part * W + wave, a.splits * W, pages, layer, exps, m, l, o);
    }

    // ---- join the waves, one column tile at a time
    extern __shared__ float shared[];  // so [W][16][D + 4], sm [16][W], sl [16][W]
    float *so = shared, *sm = so + W * 16 * (D + 4), *sl = sm + W * 16;
    constexpr int PER = D / 4;  // threads per column
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        if (x > 0) __syncthreads();
        const float inv = l[x][0] == 0.f ? 0.f : pow2(held_unit) * __builtin_amdgcn_rcpf(l[x][0]);  // averages: sums could pass fp32's range
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(so + (wave * 16 + col) * (D + 4) + 16 * d + 4 * g) = o[x][d] * inv;
        if (g == 0) {
            sm[col * W + wave] = m[x];
            sl[col * W + wave] = l[x][0];
        }
        __syncthreads();
        if (threadIdx.x < 16 * W) {  // thread (column, wave): the wave's share of the column
            const int cc = threadIdx.x / W, y = first_col + 16 * x + cc;
            const float mine = sm[threadIdx.x], top = among<W>(mine, [](float p, float q) { return fmaxf(p, q); });
            const float f = __builtin_amdgcn_exp2f(mine - (top > NEG_INF ? top : 0.f)) * sl[threadIdx.x];
            const float total = among<W>(f, [](float p, float q) { return p + q; });
            sl[threadIdx.x] = total == 0.f ? 0.f : f * __builtin_amdgcn_rcpf(total);
            if (a.splits > 1 && threadIdx.x % W == 0 && y < cs.columns) a.part_ml[(int64_t)part * a.rows + cs.row_of(y)] = make_float2(top, total);
        }
        __syncthreads();
        for (int cc = threadIdx.x / PER; cc < 16; cc += 64 * W / PER) {  // thread: column cc, four d's
            const int d = 4 * (threadIdx.x % PER);
            const int y = first_col + 16 * x + cc;
            if (y >= cs.columns) break;
            f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) v += *reinterpret_cast<const f32x4*>(so + (w * 16 + cc) * (D + 4) + d) * sl[cc * W + w];
            const int64_t r = cs.row_of(y);
            if (a.splits == 1) {
                bf16x4 b;
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = (bf16_t)v[i];
                *reinterpret_cast<bf16x4*>(a.out + r * D + d) = b;
            } else {
                *reinterpret_cast<f32x4*>(a.part_o + ((int64_t)part * a.rows + r) * D + d) = v;
            }
        }
    }
}

// Many columns (prompts): a workgroup of four waves has 128, each wave 32 of them, and all walk the same pages.  What bounds
// it is vector instructions, and a fifth of those are conversions, so every page is converted once for the four waves: each
// converts a quarter, into LDS, in the order in which the products' first operands are read (a lane's 16 bytes after
// another's: no bank conflict).  Two buffers, one barrier per page; the next page's bytes are on their way meanwhile.
// 16 prompts of up to 1541 tokens, 15 query heads on 5 of 64: 91 us (450 TFLOP/s; every wave converting for itself 105); of 4096
// tokens 735 TFLOP/s, with heads of 128 780.  Of a wave's vector issue slots 60 % are used: the rest is the prologue of short
// rows and waves of a workgroup waiting for each other.
constexpr int PROMPT_W = 4, PROMPT_CT = 2;
// (D 64: 4 waves per SIMD, a few spilled registers included, are 7 % faster than 3.)
constexpr int prompt_occupancy(int D) { return D == 64 ? 4 : 2; }
template <int D>
__global__ __launch_bounds__(64 * PROMPT_W) __attribute__((amdgpu_waves_per_eu(prompt_occupancy(D), prompt_occupancy(D))))
void kv_prompt_kernel(asrk_kv_cache c, AttnArgs a) {
    constexpr int CT = PROMPT_CT, W = PROMPT_W;
    constexpr int KS = D / 64, DT = D / 16, OWN = DT / W;  // value tiles that a wave converts
    constexpr int K_BYTES = ASRK_KV_PAGE * D * 2, BUF = 2 * K_BYTES;
    extern __shared__ __attribute__((aligned(16))) char tiles[];  // [2][keys | values]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // The last rows of every prompt first: they see the most, and what is left for the end is short.
    const int part = part_of(a), set = blockIdx.y, chunk = gridDim.z - 1 - blockIdx.z;
    const Columns cs(c, a, set);
    const int first_col = (chunk * W + wave) * 16 * CT;
    Pages work(c, a.beams, set, part, a.splits, lane);
    // How many tokens any column of the workgroup sees, of one sequence (up to its last row's own) or of each of several (lane).
    // What lies behind them in a page may not have been written yet, and may be anything.
    const int64_t seq = (int64_t)set * a.beams;
    int most, seen_of = 0;
    if (a.beams == 1) {
        const int start = c.starts[seq * c.seq_stride], fresh = c.lens[seq * c.seq_stride] - start;
        const int x0 = chunk * W * 16 * CT, x1 = x0 + W * 16 * CT < cs.columns ? x0 + W * 16 * CT : cs.columns;
        const int i0 = over(x0, a.group_inv), i1 = over(x1 - 1, a.group_inv) + 1;
        most = i0 >= fresh ? 0 : start + (i1 < fresh ? i1 : fresh);
    } else {
        if (lane < a.beams) {
            const int start = c.starts[(seq + lane) * c.seq_stride], fresh = c.lens[(seq + lane) * c.seq_stride] - start;
            seen_of = fresh <= 0 ? 0 : start + (fresh < a.n ? fresh : a.n);
        }
        most = wave_imax(seen_of);
    }
    int pages = (most + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE;
    pages = pages < c.max_pages ? pages : c.max_pages;
    if (pages <= 0) {  // nothing to see: the rows are zero
        if (a.splits == 1) {
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                const int y = first_col + 16 * x + col;
                if (y >= cs.columns) continue;
                bf16_t* p = a.out + cs.row_of(y) * D + 4 * g;
#pragma unroll
                for (int d = 0; d < DT; ++d) *reinterpret_cast<u32x2*>(p + 16 * d) = u32x2{0u, 0u};
            }
            return;
        }
    }
    Queries<D, CT> qs;
    qs.load(c, cs, first_col, col, g);

    f32x4 o[CT][DT], l[CT];
    float m[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        m[t] = NEG_INF;
        l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Unit unit;                 // of the value tiles, alike in all waves
    int held_unit = unit.now;  // of o

    const char* layer = (const char*)c.kv + a.layer * c.num_pages * cs.H * (int64_t)(2 * ASRK_KV_PAGE * D);
    const int* exps = (const int*)c.exps + a.layer * c.num_pages * cs.H;
    // this lane's bytes of the wave's quarter: keys of tile `wave`, values of tiles wave * OWN ..
    const uint32_t k_at = (16 * (col >> 2) + 4 * wave + (col & 3)) * D + 16 * g, v_at = col * ASRK_KV_PAGE + 16 * g;
    u32x4 kr[KS], vr[OWN];
    auto load_value = [&](__amdgpu_buffer_rsrc_t rows, int d) __attribute__((always_inline)) {
        return __builtin_amdgcn_raw_buffer_load_b128(rows, v_at + 16 * d * ASRK_KV_PAGE, ASRK_KV_PAGE * D, 0);
    };
    auto load_page = [&](__amdgpu_buffer_rsrc_t rows) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[s] = __builtin_amdgcn_raw_buffer_load_b128(rows, k_at + 64 * s, 0, 0);
#pragma unroll
        for (int d = 0; d < OWN; ++d)
            vr[d] = __builtin_amdgcn_raw_buffer_load_b128(rows, v_at + (wave * OWN + d) * (16 * ASRK_KV_PAGE), ASRK_KV_PAGE * D, 0);
    };
    Item item = work.next(pages);
    int64_t at = (int64_t)(item.page < 0 ? 0 : item.page) * cs.H + cs.h;
    __amdgpu_buffer_rsrc_t rows = page_rows(layer, at, D);
    char* buf = tiles;
    bool apart = false;  // alike in all waves
    if (item.page >= 0) {
        int e_next = exps[at];
        load_page(rows);
        for (;;) {
            const int e = __builtin_amdgcn_readfirstlane(e_next), ev = (int8_t)(e >> 8);
            if (__builtin_expect(!unit.follow(ev), 0)) {
                apart = true;
                break;
            }
            const int up = unit.now;
            const Item following = work.next(pages);
            at = (int64_t)(following.page < 0 ? 0 : following.page) * cs.H + cs.h;
            const __amdgpu_buffer_rsrc_t rows_next = page_rows(layer, at, D);
            if (following.page >= 0) e_next = exps[at];
            const bool odd = __builtin_expect((e >> 16) & 1, 0);
            {
                const float ks = pow2((int8_t)e), vs = pow2(ev - up);
                const int last = (a.beams == 1 ? most : wave_imax((item.with >> lane) & 1 ? seen_of : 0)) - item.p * ASRK_KV_PAGE;
                if (last < ASRK_KV_PAGE) {  // within the page
                    KEEP_BRANCH();
                    const u32x4 mask = keep_before(last, g);
#pragma unroll
                    for (int d = 0; d < OWN; ++d) vr[d] &= mask;
                }
                if (odd) {
                    KEEP_BRANCH();
#pragma unroll
                    for (int d = 0; d < OWN; ++d)
#pragma unroll
                        for (int w = 0; w < 4; ++w) vr[d][w] &= ~nan_bytes(vr[d][w]);
                }
                // fragment (tile, step): 64 lanes of 16 bytes
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    bf16x8* to = reinterpret_cast<bf16x8*>(buf) + (wave * 2 * KS + 2 * s) * 64 + lane;
                    to[0] = k8(kr[s][0], kr[s][1], ks);
                    to[64] = k8(kr[s][2], kr[s][3], ks);
                }
#pragma unroll
                for (int d = 0; d < OWN; ++d) {
                    f16x8* to = reinterpret_cast<f16x8*>(buf + K_BYTES) + (wave * OWN + d) * 128 + lane;
                    to[0] = v8(vr[d][0], vr[d][1], vs);
                    to[64] = v8(vr[d][2], vr[d][3], vs);
                }
            }
            __syncthreads();  // the other buffer was last read before the barrier in front of this one
            if (following.page >= 0) load_page(rows_next);
            int seen[CT];
            bool whole;
            if (qs.see(item.p, item.with, seen, whole)) {
                const bf16x8* kt = reinterpret_cast<const bf16x8*>(buf) + lane;
                const f16x8* vt = reinterpret_cast<const f16x8*>(buf + K_BYTES) + lane;
                f32x4 sc[CT][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int x = 0; x < CT; ++x) sc[x][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < 2 * KS; ++s) {
                        const bf16x8 k = kt[(t * 2 * KS + s) * 64];
#pragma unroll
                        for (int x = 0; x < CT; ++x) sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qs.q[x][s], sc[x][t], 0, 0, 0);
                    }
                }
                f16x8 pf[CT][2];
                weigh<CT, DT>(sc, seen, whole, g, a.c, up, held_unit, m, l, o, pf);
                held_unit = up;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const f16x8 v = vt[(d * 2 + u) * 64];
#pragma unroll
                        for (int x = 0; x < CT; ++x) o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[x][u], o[x][d], 0, 0, 0);
                    }
                add_weights<CT>(pf, l);
                if (odd) mark_nans<CT, DT>([&](int d) { return load_value(rows, d); }, seen, g, o);
            }
            buf = buf == tiles ? tiles + BUF : tiles;
            if (following.page < 0) break;
            item = following;
            rows = rows_next;
        }
    }
    if (__builtin_expect(apart, 0)) {
        held_unit = APART;
        walk_apart_anew<D, CT>(c, cs, first_col, part, a.splits, pages, layer, exps, m, l, o);
    }
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        const int y = first_col + 16 * x + col;
        if (y >= cs.columns) continue;
        const int64_t r = cs.row_of(y);
        const float inv = l[x][0] == 0.f ? 0.f : pow2(held_unit) * __builtin_amdgcn_rcpf(l[x][0]);
        if (a.splits == 1) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                bf16x4 b;
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = (bf16_t)(o[x][d][i] * inv);
                *reinterpret_cast<bf16x4*>(a.out + r * D + 16 * d + 4 * g) = b;
            }
        } else {
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(a.part_o + ((int64_t)part * a.rows + r) * D + 16 * d + 4 * g) = o[x][d] * inv;
            if (g == 0) a.part_ml[(int64_t)part * a.rows + r] = make_float2(m[x], l[x][0]);
        }
    }
}

// Joins the splits (averages, with their maxima and sums of weights): D / 4 lanes per row.
template <int D>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, int splits,
                                                                int64_t rows, bf16_t* __restrict__ out) {
    const int64_t r = (int64_t)blockIdx.x * (1024 / D) + threadIdx.x / (D / 4);
    const int d = threadIdx.x % (D / 4) * 4;
    if (r >= rows) return;
    float top = NEG_INF;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) top = fmaxf(top, part_ml[s * rows + r].x);
    const float ref = top > NEG_INF ? top : 0.f;
    float total = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float2 ml = part_ml[s * rows + r];
        total += __builtin_amdgcn_exp2f(ml.x - ref) * ml.y;
    }
    const float share = total == 0.f ? 0.f : 1.f / total;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float2 ml = part_ml[s * rows + r];
        v += *reinterpret_cast<const f32x4*>(part_o + (s * rows + r) * D + d) * (__builtin_amdgcn_exp2f(ml.x - ref) * ml.y * share);
    }
    bf16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (bf16_t)v[i];
    *reinterpret_cast<bf16x4*>(out + r * D + d) = y;
}

struct Plan {
    int ct, waves, splits, chunks;
    bool prompt;
};
// By the capacity of the table, not by the lengths, which only the device knows.
//  - 128 columns or more: kv_prompt_kernel.
//  - Fewer: the waves of a workgroup share them and deal the pages.  Up to 48 pages one workgroup does it all: a second
//    launch to join splits costs 4 us, more than it saves (5 beams over 26 pages, 5 heads: 11.9 us, in 4 splits 15.8;
//    64 times that: 19.6, in 2 splits 27.8).  Beyond, enough splits for 1024 workgroups, of two pages per wave at least
//    (48 sequences, 8 heads of 128, 256 pages: 213 us unsplit, 204 in 2, 201 in 3).
Plan plan_of(const asrk_kv_cache* c, int n, int q_heads, int beams) {
    const int64_t columns = (int64_t)beams * n * (q_heads / c->kv_heads);
    Plan p;
    p.prompt = columns >= 128;
    p.ct = columns > 16 ? 2 : 1;
    p.waves = p.prompt || p.ct == 2 ? 4 : 8;
    const int per = 16 * p.ct * (p.prompt ? p.waves : 1);
    p.chunks = (int)((columns + per - 1) / per);
    p.splits = 1;
    const int64_t groups = (int64_t)c->kv_heads * (c->num_seqs / beams) * p.chunks;
    const int64_t want = ((p.prompt ? 512 : 1024) + groups - 1) / groups, most = c->max_pages / (p.prompt ? 16 : 2 * p.waves);
    if (c->max_pages > 48) {
        p.splits = (int)(want < most ? want : most);
        if (p.splits > 128) p.splits = 128;
    }
    return p;
}

template <class K>
int launch(K kernel, const asrk_kv_cache* c, const AttnArgs& a, int threads, int lds, int chunks, std::atomic<uint64_t>& done, hipStream_t st) {
    if (lds > 60000)  // beside what the kernel declares itself, 64 KiB need asking for
        if (int rc = asrk_max_lds_once((const void*)kernel, lds, done)) return rc;
    hipLaunchKernelGGL(kernel, dim3(c->kv_heads * a.splits, c->num_seqs / a.beams, chunks), dim3(threads), lds, st, *c, a);
    return ASRK_OK;
}
template <int D, int CT, int W>
int launch_shared(const asrk_kv_cache* c, const AttnArgs& a, int chunks, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    return launch(kv_attention_kernel<D, CT, W>, c, a, 64 * W, (W * 16 * (D + 4) + 2 * W * 16) * (int)sizeof(float), chunks, done, st);
}
template <int D>
int launch_for(const asrk_kv_cache* c, const AttnArgs& a, const Plan& p, hipStream_t st) {
    if (p.prompt) {
        static std::atomic<uint64_t> done{0};
        return launch(kv_prompt_kernel<D>, c, a, 64 * PROMPT_W, 4 * ASRK_KV_PAGE * D * 2, p.chunks, done, st);
    }
    return p.ct == 2 ? launch_shared<D, 2, 4>(c, a, p.chunks, st) : launch_shared<D, 1, 8>(c, a, p.chunks, st);
}

int check_shape(const asrk_kv_cache* c, int n, int q_heads, int beams) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (n <= 0 || q_heads <= 0 || q_heads % c->kv_heads || beams <= 0 || beams > 32 || c->num_seqs % beams) return ASRK_ERR_SHAPE;
    if ((int64_t)beams * n * (q_heads / c->kv_heads) > 65535 * 128) return ASRK_ERR_SHAPE;  // the grid's last dimension
    return ASRK_OK;
}

}  // namespace

extern "C" size_t asrk_kv_attention_workspace_bytes(const asrk_kv_cache* c, int n, int q_heads, int num_beams) {
    if (check_shape(c, n, q_heads, num_beams)) return 0;
    const Plan p = plan_of(c, n, q_heads, num_beams);
    return p.splits == 1 ? 0 : (size_t)p.splits * c->num_seqs * n * q_heads * (c->head_dim * sizeof(float) + sizeof(float2));
}

extern "C" int asrk_kv_attention(const asrk_kv_cache* c, int layer, const void* q, int64_t seq_ld, int64_t row_ld, int64_t head_ld, int n,
                                 int q_heads, int num_beams, float scale, void* out, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_shape(c, n, q_heads, num_beams)) return rc;
    if (!q || !out) return ASRK_ERR_NULL;
    if (layer < 0 || layer >= c->num_layers || seq_ld < 0 || row_ld < 0 || head_ld < 0 || !(scale > 0.f && scale < 1e30f)) return ASRK_ERR_SHAPE;
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || seq_ld % 8 || row_ld % 8 || head_ld % 8) return ASRK_ERR_ALIGN;
    const Plan p = plan_of(c, n, q_heads, num_beams);
    const int64_t rows = (int64_t)c->num_seqs * n * q_heads;
    AttnArgs a{};
    if (p.splits > 1) {
        if (!ws) return ASRK_ERR_NULL;
        if ((uintptr_t)ws & 15) return ASRK_ERR_ALIGN;
        if (ws_bytes < asrk_kv_attention_workspace_bytes(c, n, q_heads, num_beams)) return ASRK_ERR_WORKSPACE;
        a.part_o = (float*)ws;
        a.part_ml = (float2*)((char*)ws + (size_t)p.splits * rows * c->head_dim * sizeof(float));
    }
    a.q = (const bf16_t*)q;
    a.out = (bf16_t*)out;
    a.seq_ld = seq_ld;
    a.row_ld = row_ld;
    a.head_ld = head_ld;
    a.layer = layer;
    a.rows = rows;
    a.n = n;
    a.group = q_heads / c->kv_heads;
    a.beams = num_beams;
    a.splits = p.splits;
    a.per_seq_inv = 1.0 / ((double)n * a.group);
    a.group_inv = 1.0 / a.group;
    a.c = scale * 1.4426950408889634f;
    hipStream_t st = (hipStream_t)stream;
    if (int rc = c->head_dim == 64 ? launch_for<64>(c, a, p, st) : launch_for<128>(c, a, p, st)) return rc;
    if (p.splits > 1) {
        const int per = 1024 / c->head_dim;
        const dim3 grid((unsigned)((rows + per - 1) / per));
        if (c->head_dim == 64)
            hipLaunchKernelGGL(kv_attention_join_kernel<64>, grid, dim3(256), 0, st, a.part_o, a.part_ml, p.splits, rows, a.out);
        else
            hipLaunchKernelGGL(kv_attention_join_kernel<128>, grid, dim3(256), 0, st, a.part_o, a.part_ml, p.splits, rows, a.out);
    }
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}
