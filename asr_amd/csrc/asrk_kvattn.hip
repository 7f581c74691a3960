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
// Keys become bf16 with their scale applied (exact); values become f16 in units of 2^E, E the largest exponent so far:
// exact up to a ratio of 2^15 between pages, below that to 2^-25 of the largest value.  Weights are rounded to f16, 2^-11
// relative, 8 times finer than bf16 would be and well under the 2^-8 of the bf16 result.  Everything else is fp32.
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
    int64_t seq_ld, row_ld, head_ld, layer;
    int n, group, beams, splits;  // new tokens, query heads per key/value head
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
__device__ __forceinline__ int wave_imax(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int y = __shfl_xor(v, o, 64);
        v = v > y ? v : y;
    }
    return v;
}

// Waves per SIMD that the registers are cut for: as many as hold a page, q, o and the scores without spilling in the loop.
// (D 64, 1 tile: 4; with 3, 64 x 5 beams take 24.5 us instead of 19.7.  D 128, 1 tile: 2; with 3 it spills and 1.2 GB of
// cache take 228 us instead of 204.)
constexpr int occupancy(int D, int CT) { return D == 64 ? (CT == 1 ? 4 : 3) : 2; }

// CT column tiles of 16 per wave.  OWN_COLUMNS: every wave has columns of its own and walks all pages (prompts, where
// columns abound); otherwise the W waves share the columns and deal the pages among them (and among the splits).
template <int D, int CT, int W, bool OWN_COLUMNS>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(occupancy(D, CT), occupancy(D, CT))))
void kv_attention_kernel(asrk_kv_cache c, AttnArgs a) {
    constexpr int KS = D / 64;   // 16-byte pieces of a key row per lane
    constexpr int DT = D / 16;   // tiles of 16 d
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int H = c.kv_heads, M = c.max_pages;
    const int h = blockIdx.y;
    const int per_seq = a.n * a.group;          // columns of a sequence
    const int columns = a.beams * per_seq;
    const int chunks = (columns + 16 * CT * (OWN_COLUMNS ? W : 1) - 1) / (16 * CT * (OWN_COLUMNS ? W : 1));
    // The last rows of every prompt first: they see the most, and what is left for the end is short.
    const int sets = c.num_seqs / a.beams, set = blockIdx.z % sets, chunk = chunks - 1 - blockIdx.z / sets;
    const int first_col = (OWN_COLUMNS ? chunk * W + wave : chunk) * 16 * CT;

    // The pages of a wave: by its number alone, so that their numbers are on the way before the lengths are known.
    const int p0 = OWN_COLUMNS ? 0 : blockIdx.x * W + wave, step = OWN_COLUMNS ? 1 : a.splits * W;
    const int* table = c.table + ((int64_t)set * a.beams + lane) * c.seq_stride * M;  // of beam `lane`
    auto page_of = [&](int p) __attribute__((always_inline)) { return lane < a.beams && p < M ? table[p] : -1; };
    int coming = page_of(p0);

    auto split = [&](int y, int& b, int& i, int& j) __attribute__((always_inline)) {  // column: beam, new token, query head
        b = a.beams == 1 ? 0 : (int)((unsigned)y / (unsigned)per_seq);
        const unsigned in = (unsigned)(y - b * per_seq);
        i = a.n == 1 ? 0 : (int)(in / (unsigned)a.group);
        j = (int)in - i * a.group;
    };
    auto row_of = [&](int y) __attribute__((always_inline)) {  // of q and out, in units of D
        int b, i, j;
        split(y, b, i, j);
        return (((int64_t)set * a.beams + b) * a.n + i) * (int64_t)(H * a.group) + h * a.group + j;
    };
    // ---- this lane's columns: beam, tokens seen, row of q
    int limit[CT], beam[CT];
    bf16x8 qf[CT][2 * KS];
    int most = 0;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int x = first_col + 16 * t + col;
        int b, i, j;
        split(x, b, i, j);
        beam[t] = 0;
        limit[t] = NO_COLUMN;
#pragma unroll
        for (int s = 0; s < 2 * KS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) qf[t][s][e] = (bf16_t)0.f;
        if (x < columns) {
            const int64_t seq = (int64_t)set * a.beams + b;
            const int start = c.starts[seq * c.seq_stride], fresh = c.lens[seq * c.seq_stride] - start;
            beam[t] = b;
            limit[t] = i >= fresh ? 0 : (start + i + 1 < M * ASRK_KV_PAGE ? start + i + 1 : M * ASRK_KV_PAGE);
            most = limit[t] > most ? limit[t] : most;
            const bf16_t* q = a.q + seq * a.seq_ld + (int64_t)i * a.row_ld + (int64_t)(h * a.group + j) * a.head_ld + 16 * g;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[t][2 * s] = *reinterpret_cast<const bf16x8*>(q + 64 * s);
                qf[t][2 * s + 1] = *reinterpret_cast<const bf16x8*>(q + 64 * s + 8);
            }
        }
    }
    most = __builtin_amdgcn_readfirstlane(wave_imax(most));

    f32x4 o[CT][DT], l[CT];
    float m[CT];
    const f16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        m[t] = NEG_INF;
        l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int unit = ASRK_KV_EXP_MIN;  // o is in units of 2^unit

    const int pages = (most + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE;
    const char* layer = (const char*)c.kv + a.layer * c.num_pages * H * (int64_t)(2 * ASRK_KV_PAGE * D);
    const int* exps = (const int*)c.exps + a.layer * c.num_pages * H;
    const uint32_t k_at = (16 * (col >> 2) + (col & 3)) * D + 16 * g, v_at = col * ASRK_KV_PAGE + 16 * g;  // this lane's bytes

    // The wave's work, page by page: beams whose tables agree on a page take it together.
    struct Item {
        int page, p;  // -1: no more; the p-th page of its sequences
        uint64_t with;
    };
    int at_p = p0, item_p = 0, mine = -1;
    uint64_t left = 0;
    auto advance = [&]() __attribute__((always_inline)) -> Item {
        while (!left) {
            if (at_p >= pages) return Item{-1, 0, 0};
            mine = coming;
            item_p = at_p;
            at_p += step;
            coming = page_of(at_p);
            left = __ballot(mine >= 0 && mine < c.num_pages);
        }
        const int page = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t with = __ballot(mine == page) & left;
        left &= ~with;
        return Item{page, item_p, with};
    };
    // Loads go through a descriptor of the page: one register of lane offset, the rest in the instruction.
    auto rows_of = [&](int page) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform_ptr(layer + ((int64_t)page * H + h) * (2 * ASRK_KV_PAGE * D))), 0,
                                                 2 * ASRK_KV_PAGE * D, 0x00020000);
    };
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
    Item item = advance();
    __amdgpu_buffer_rsrc_t rows = rows_of(item.page < 0 ? 0 : item.page);
    int e_next = 0;
    if (item.page >= 0) {
        e_next = exps[(int64_t)item.page * H + h];
        load_keys(rows);
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[d] = load_value(rows, d);
    }
    while (item.page >= 0) {
        // The next page's keys are loaded over this one's as soon as the scores are done, its values as soon as they are used.
        const Item following = advance();
        const __amdgpu_buffer_rsrc_t rows_next = rows_of(following.page < 0 ? 0 : following.page);
        {
            const int p = item.p;
            const uint64_t with = item.with;
            const int e = __builtin_amdgcn_readfirstlane(e_next);
            if (following.page >= 0) e_next = exps[(int64_t)following.page * H + h];
            // ---- which columns see how much of it
            int seen[CT];
            int all = ASRK_KV_PAGE, some = 0;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int s = limit[t] - p * ASRK_KV_PAGE;
                const bool takes = (with >> beam[t]) & 1;
                seen[t] = limit[t] == NO_COLUMN || (takes && s > ASRK_KV_PAGE) ? ASRK_KV_PAGE : (takes && s > 0 ? s : 0);
                all = seen[t] < all ? seen[t] : all;
                some = seen[t] > some && limit[t] != NO_COLUMN ? seen[t] : some;
            }
            const bool whole = __all(all == ASRK_KV_PAGE);

            const float ks = pow2((int8_t)e);
            const int ev = (int8_t)(e >> 8);
            // ---- scores
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
                        sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[x][2 * s], sc[x][t], 0, 0, 0);
                        sc[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[x][2 * s + 1], sc[x][t], 0, 0, 0);
                    }
                }
            }
            if (following.page >= 0) load_keys(rows_next);
            // ---- weights
            // The reference follows the maximum only when that has grown by more than 2^8: up to there the weights stay
            // within f16, at the same relative precision, and o and the sum need no rescaling.
            const int up = ev > unit ? ev : unit;
            const float shrink = pow2(unit - up);
            f16x8 pf[CT][2];
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
                const float now = groups_max(top) * a.c;  // c > 0
                if (__any(now > m[x] + 8.f) || up != unit) {
                    KEEP_BRANCH();
                    const float to = now > m[x] + 8.f ? now : m[x];  // by the column alone: its bits do not depend on its neighbours
                    const float back = to > NEG_INF ? __builtin_amdgcn_exp2f(m[x] - to) : 0.f;
                    m[x] = to;
#pragma unroll
                    for (int i = 0; i < 4; ++i) l[x][i] *= back;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[x][d] *= back * shrink;
                }
                const float ref = m[x] > NEG_INF ? m[x] : 0.f;  // nothing seen yet: every weight is 0
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const f32x2_t w = {__builtin_amdgcn_exp2f(fmaf(sc[x][t][i], a.c, -ref)),
                                           __builtin_amdgcn_exp2f(fmaf(sc[x][t][i + 1], a.c, -ref))};
                        const f16x2 h = __builtin_convertvector(w, f16x2);  // to nearest
                        pf[x][t >> 1][4 * (t & 1) + i] = h[0];
                        pf[x][t >> 1][4 * (t & 1) + i + 1] = h[1];
                    }
            }
            unit = up;
            const float vs = pow2(ev - up);
            if (!whole) {  // bytes behind the last token seen by anyone may be anything
                KEEP_BRANCH();
                const int last = wave_imax(some) - 16 * g;
                uint32_t mask[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int keep = last - 4 * w < 0 ? 0 : (last - 4 * w > 4 ? 4 : last - 4 * w);
                    mask[w] = (uint32_t)((1ull << (8 * keep)) - 1);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        vr[d][w] &= mask[w];
                    }
            }
            // The values may hold a NaN (rare: the page says so), and 0 * NaN must not reach columns that do not see its
            // token.  The NaNs become zeros, and below, what a product of the 0/1 patterns (is a NaN, is seen) says becomes NaN.
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
            // the sum of the weights as they are used: a product with ones, all four rows of a lane are the column's sum
#pragma unroll
            for (int x = 0; x < CT; ++x)
#pragma unroll
                for (int u = 0; u < 2; ++u) l[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[x][u], l[x], 0, 0, 0);
            if (odd) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    __builtin_amdgcn_sched_barrier(0);  // one tile at a time: this path must not cost the other one registers
                    const u32x4 raw = load_value(rows, d);
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
        }
        if (following.page >= 0) {
#pragma unroll
            for (int d = 0; d < DT; ++d) vr[d] = load_value(rows_next, d);
        }
        item = following;
        rows = rows_next;
    }
    if (OWN_COLUMNS) {
#pragma unroll
        for (int x = 0; x < CT; ++x) {
            const int y = first_col + 16 * x + col;
            if (y >= columns) continue;
            const int64_t r = row_of(y);
            const float inv = l[x][0] == 0.f ? 0.f : pow2(unit) / l[x][0];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                bf16x4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (bf16_t)(o[x][d][i] * inv);
                *reinterpret_cast<bf16x4*>(a.out + r * D + 16 * d + 4 * g) = y;
            }
        }
        return;
    }
    // ---- join the waves, one column tile at a time: thread: column cc, four d's from dd on
    extern __shared__ float shared[];  // so [W][16][D + 4], sm [W][16], sl [W][16]
    float *so = shared, *sm = so + W * 16 * (D + 4), *sl = sm + W * 16;
    constexpr int PER = D / 4;  // threads per column
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        if (x > 0) __syncthreads();
        const float u = pow2(unit);
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(so + (wave * 16 + col) * (D + 4) + 16 * d + 4 * g) = o[x][d] * u;
        if (g == 0) {
            sm[wave * 16 + col] = m[x];
            sl[wave * 16 + col] = l[x][0];
        }
        __syncthreads();
        for (int cc = threadIdx.x / PER; cc < 16; cc += 64 * W / PER) {
            const int d = 4 * (threadIdx.x % PER);
            const int y = first_col + 16 * x + cc;
            if (y >= columns) break;
            float top = NEG_INF;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w * 16 + cc]);
            const float ref = top > NEG_INF ? top : 0.f;
            float total = 0.f;
            f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm[w * 16 + cc] - ref);
                total += f * sl[w * 16 + cc];
                v += *reinterpret_cast<const f32x4*>(so + (w * 16 + cc) * (D + 4) + d) * f;
            }
            const int64_t r = row_of(y);
            const int64_t rows = (int64_t)c.num_seqs * a.n * H * a.group;
            if (a.splits == 1) {
                const float inv = total == 0.f ? 0.f : 1.f / total;
                bf16x4 b;
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = (bf16_t)(v[i] * inv);
                *reinterpret_cast<bf16x4*>(a.out + r * D + d) = b;
            } else {
                *reinterpret_cast<f32x4*>(a.part_o + ((int64_t)blockIdx.x * rows + r) * D + d) = v;
                if (d == 0) a.part_ml[(int64_t)blockIdx.x * rows + r] = make_float2(top, total);
            }
        }
    }
}

// Joins the splits: D / 4 lanes per row.
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
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float2 ml = part_ml[s * rows + r];
        const f32x4 part = *reinterpret_cast<const f32x4*>(part_o + (s * rows + r) * D + d);
        const float f = __builtin_amdgcn_exp2f(ml.x - ref);
        total += f * ml.y;
        v += part * f;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    bf16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (bf16_t)(v[i] * inv);
    *reinterpret_cast<bf16x4*>(out + r * D + d) = y;
}

struct Plan {
    int ct, waves, splits, chunks;
    bool own;
};
// By the capacity of the table, not by the lengths, which only the device knows.
//  - 128 columns or more: four waves with columns of their own, each over all pages.
//  - Fewer: the waves of a workgroup share them and deal the pages.  Up to 48 pages one workgroup does it all: a second
//    launch to join splits costs 4 us, more than it saves (5 beams over 26 pages, 5 heads: 11.9 us, in 4 splits 15.8;
//    64 times that: 19.6, in 2 splits 27.8).  Beyond, enough splits for 1024 workgroups, of two pages per wave at least
//    (48 sequences, 8 heads of 128, 256 pages: 213 us unsplit, 204 in 2, 201 in 3).
Plan plan_of(const asrk_kv_cache* c, int n, int q_heads, int beams) {
    const int64_t columns = (int64_t)beams * n * (q_heads / c->kv_heads);
    Plan p;
    p.own = columns >= 128;
    p.ct = columns > 16 ? 2 : 1;
    p.waves = p.own || p.ct == 2 ? 4 : 8;
    const int per = 16 * p.ct * (p.own ? p.waves : 1);
    p.chunks = (int)((columns + per - 1) / per);
    p.splits = 1;
    if (!p.own && c->max_pages > 48) {
        const int64_t groups = (int64_t)c->kv_heads * (c->num_seqs / beams) * p.chunks;
        const int64_t want = (1024 + groups - 1) / groups, most = c->max_pages / (2 * p.waves);
        p.splits = (int)(want < most ? want : most);
        if (p.splits > 128) p.splits = 128;
    }
    return p;
}

template <int D, int CT, int W, bool OWN>
int launch(const asrk_kv_cache* c, const AttnArgs& a, int sets, int chunks, hipStream_t st) {
    constexpr int lds = OWN ? 0 : (W * 16 * (D + 4) + 2 * W * 16) * (int)sizeof(float);
    if (lds > 65536) {
        static std::atomic<uint64_t> done{0};
        if (int rc = asrk_max_lds_once((const void*)kv_attention_kernel<D, CT, W, OWN>, lds, done)) return rc;
    }
    hipLaunchKernelGGL((kv_attention_kernel<D, CT, W, OWN>), dim3(a.splits, c->kv_heads, sets * chunks), dim3(64 * W), lds, st, *c, a);
    return ASRK_OK;
}
template <int D>
int launch_for(const asrk_kv_cache* c, const AttnArgs& a, const Plan& p, int sets, hipStream_t st) {
    if (p.own) return launch<D, 2, 4, true>(c, a, sets, p.chunks, st);
    if (p.ct == 2) return launch<D, 2, 4, false>(c, a, sets, p.chunks, st);
    return launch<D, 1, 8, false>(c, a, sets, p.chunks, st);
}

int check_shape(const asrk_kv_cache* c, int n, int q_heads, int beams) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (n <= 0 || q_heads <= 0 || q_heads % c->kv_heads || beams <= 0 || beams > 32 || c->num_seqs % beams) return ASRK_ERR_SHAPE;
    if ((int64_t)beams * n * (q_heads / c->kv_heads) > 0x3fffffff) return ASRK_ERR_SHAPE;
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
    if (layer < 0 || layer >= c->num_layers || seq_ld < 0 || row_ld < 0 || head_ld < 0 || !(scale > 0.f)) return ASRK_ERR_SHAPE;
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || seq_ld % 8 || row_ld % 8 || head_ld % 8) return ASRK_ERR_ALIGN;
    const Plan p = plan_of(c, n, q_heads, num_beams);
    const int sets = c->num_seqs / num_beams;
    if ((int64_t)sets * p.chunks > 65535) return ASRK_ERR_SHAPE;
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
    a.n = n;
    a.group = q_heads / c->kv_heads;
    a.beams = num_beams;
    a.splits = p.splits;
    a.c = scale * 1.4426950408889634f;
    hipStream_t st = (hipStream_t)stream;
    if (int rc = c->head_dim == 64 ? launch_for<64>(c, a, p, sets, st) : launch_for<128>(c, a, p, sets, st)) return rc;
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
