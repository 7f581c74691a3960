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

constexpr int WAVES = 4;
constexpr int NO_COLUMN = 0x7fffffff;  // limit of a lane behind the last column: takes part in nothing, and masks nothing
constexpr float NEG_INF = -__builtin_inff();

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

// Maximum over the lanes of a column's four groups, and over all lanes of a wave.
__device__ __forceinline__ float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ int wave_imax(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int y = __shfl_xor(v, o, 64);
        v = v > y ? v : y;
    }
    return v;
}

// CT column tiles of 16 per wave.  OWN_COLUMNS: every wave has columns of its own and walks all pages (prompts, where
// columns abound); otherwise the four waves share the columns and deal the pages of the workgroup's split among them.
template <int D, int CT, bool OWN_COLUMNS>
__global__ __launch_bounds__(256) void kv_attention_kernel(asrk_kv_cache c, AttnArgs a) {
    constexpr int KS = D / 64;   // 16-byte pieces of a key row per lane
    constexpr int DT = D / 16;   // tiles of 16 d
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int H = c.kv_heads, M = c.max_pages;
    const int h = blockIdx.y;
    const int per_seq = a.n * a.group;          // columns of a sequence
    const int columns = a.beams * per_seq;
    const int chunks = (columns + 16 * CT * (OWN_COLUMNS ? WAVES : 1) - 1) / (16 * CT * (OWN_COLUMNS ? WAVES : 1));
    const int set = blockIdx.z / chunks, chunk = blockIdx.z % chunks;
    const int first_col = (OWN_COLUMNS ? chunk * WAVES + wave : chunk) * 16 * CT;

    // ---- this lane's columns: beam, tokens seen, row of q
    int limit[CT], beam[CT];
    int64_t row[CT];  // of out, -1: none
    bf16x8 qf[CT][2 * KS];
    int most = 0;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int x = first_col + 16 * t + col;
        const int b = x / per_seq, i = x % per_seq / a.group, j = x % a.group;
        beam[t] = 0;
        limit[t] = NO_COLUMN;
        row[t] = -1;
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
            row[t] = (seq * a.n + i) * (int64_t)(H * a.group) + h * a.group + j;
            const bf16_t* q = a.q + seq * a.seq_ld + (int64_t)i * a.row_ld + (int64_t)(h * a.group + j) * a.head_ld + 16 * g;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[t][2 * s] = *reinterpret_cast<const bf16x8*>(q + 64 * s);
                qf[t][2 * s + 1] = *reinterpret_cast<const bf16x8*>(q + 64 * s + 8);
            }
        }
    }
    most = __builtin_amdgcn_readfirstlane(wave_imax(most));

    f32x4 o[CT][DT];
    float m[CT], l[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        m[t] = NEG_INF;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int unit = ASRK_KV_EXP_MIN;  // o is in units of 2^unit

    const int pages = (most + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE;
    int p0 = 0, p1 = pages, step = 1;
    if (!OWN_COLUMNS) {
        const int per = (pages + a.splits - 1) / a.splits;
        p0 = blockIdx.x * per;
        p1 = p0 + per < pages ? p0 + per : pages;
        p0 += wave;
        step = WAVES;
    }
    const char* layer = (const char*)c.kv + a.layer * c.num_pages * H * (int64_t)(2 * ASRK_KV_PAGE * D);
    const int* exps = (const int*)c.exps + a.layer * c.num_pages * H;
    const int* table = c.table + (int64_t)set * a.beams * c.seq_stride * M;

    for (int p = p0; p < p1; p += step) {
        // Beams whose tables agree on this page take it together.
        int mine = -1;
        if (lane < a.beams) mine = table[(int64_t)lane * c.seq_stride * M + p];
        uint64_t left = __ballot(mine >= 0 && mine < c.num_pages);
        while (left) {
            const int page = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
            const uint64_t with = __ballot(mine == page) & left;
            left &= ~with;
            // ---- which columns see how much of it
            int seen[CT];
            int all = ASRK_KV_PAGE, some = 0;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int s = limit[t] - p * ASRK_KV_PAGE;
                seen[t] = limit[t] == NO_COLUMN || ((with >> beam[t]) & 1 && s > ASRK_KV_PAGE) ? ASRK_KV_PAGE : ((with >> beam[t]) & 1 ? s : 0);
                all = seen[t] < all ? seen[t] : all;
                some = seen[t] > some && limit[t] != NO_COLUMN ? seen[t] : some;
            }
            if (!__any(some > 0)) continue;
            const bool whole = __all(all == ASRK_KV_PAGE);

            const int64_t at = (int64_t)page * H + h;
            const char* kp = layer + at * (2 * ASRK_KV_PAGE * D);
            const char* vp = kp + ASRK_KV_PAGE * D;
            const int e = __builtin_amdgcn_readfirstlane(exps[at]);
            u32x4 kr[4][KS], vr[DT];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    kr[t][s] = *reinterpret_cast<const u32x4*>(kp + (16 * (col >> 2) + 4 * t + (col & 3)) * D + 64 * s + 16 * g);
#pragma unroll
            for (int d = 0; d < DT; ++d) vr[d] = *reinterpret_cast<const u32x4*>(vp + (16 * d + col) * ASRK_KV_PAGE + 16 * g);

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
            // ---- weights
            const int up = ev > unit ? ev : unit;
            const float shrink = pow2(unit - up);
            f16x8 pf[CT][2];
#pragma unroll
            for (int x = 0; x < CT; ++x) {
                float top = NEG_INF;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = sc[x][t][i] * a.c;
                        if (!whole) v = 16 * g + 4 * t + i < seen[x] ? v : NEG_INF;
                        sc[x][t][i] = v;
                        top = fmaxf(top, v);
                    }
                const float now = fmaxf(m[x], groups_max(top));
                const float ref = now > NEG_INF ? now : 0.f;  // nothing seen yet: every weight is 0
                const float back = __builtin_amdgcn_exp2f(m[x] - ref) * shrink;
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = __builtin_amdgcn_exp2f(sc[x][t][i] - ref);
                        sum += w;
                        pf[x][t >> 1][4 * (t & 1) + i] = (_Float16)w;
                    }
                l[x] = l[x] * __builtin_amdgcn_exp2f(m[x] - ref) + sum;
                m[x] = now;
                if (!__all(back == 1.f)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[x][d] *= back;
                }
            }
            unit = up;
            const float vs = pow2(ev - up);
            if (!whole) {  // bytes behind the last token seen by anyone may be anything
                const int last = wave_imax(some) - 16 * g;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int keep = last - 4 * w;
                        vr[d][w] &= keep >= 4 ? 0xffffffffu : (keep <= 0 ? 0u : (1u << (8 * keep)) - 1u);
                    }
            }
            if (__builtin_expect((e >> 16) & 1, 0)) {
                // The values hold a NaN: 0 * NaN must not reach columns that do not see its token.  Multiply without the
                // NaNs, then make NaN what a product of the two 0/1 patterns (is a NaN, is seen) says.
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f16x8 v = v8(vr[d][2 * u], vr[d][2 * u + 1], vs), bad;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const bool is = v[i] != v[i];
                            bad[i] = is ? (_Float16)1.f : (_Float16)0.f;
                            v[i] = is ? (_Float16)0.f : v[i];
                        }
#pragma unroll
                        for (int x = 0; x < CT; ++x) {
                            f16x8 sees;
#pragma unroll
                            for (int i = 0; i < 8; ++i) sees[i] = 16 * g + 8 * u + i < seen[x] ? (_Float16)1.f : (_Float16)0.f;
                            o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[x][u], o[x][d], 0, 0, 0);
                            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, sees, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[x][d][i] = hit[i] > 0.f ? __builtin_nanf("") : o[x][d][i];
                        }
                    }
            } else {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const f16x8 v = v8(vr[d][2 * u], vr[d][2 * u + 1], vs);
#pragma unroll
                        for (int x = 0; x < CT; ++x) o[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pf[x][u], o[x][d], 0, 0, 0);
                    }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        l[x] += __shfl_xor(l[x], 16, 64);
        l[x] += __shfl_xor(l[x], 32, 64);
    }

    if (OWN_COLUMNS) {
#pragma unroll
        for (int x = 0; x < CT; ++x) {
            if (row[x] < 0) continue;
            const float inv = l[x] == 0.f ? 0.f : pow2(unit) / l[x];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                bf16x4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (bf16_t)(o[x][d][i] * inv);
                *reinterpret_cast<bf16x4*>(a.out + row[x] * D + 16 * d + 4 * g) = y;
            }
        }
        return;
    }
    // ---- join the four waves, one column tile at a time
    __shared__ float so[WAVES][16][D + 4];
    __shared__ float sm[WAVES][16], sl[WAVES][16];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
        if (x > 0) __syncthreads();
        const float u = pow2(unit);
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&so[wave][col][16 * d + 4 * g]) = o[x][d] * u;
        if (g == 0) {
            sm[wave][col] = m[x];
            sl[wave][col] = l[x];
        }
        __syncthreads();
        // thread: column threadIdx.x / 16, d = 4 (threadIdx.x % 16) + 64 k
        const int cc = threadIdx.x >> 4;
        float top = NEG_INF;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w][cc]);
        const float ref = top > NEG_INF ? top : 0.f;
        float f[WAVES], total = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            f[w] = __builtin_amdgcn_exp2f(sm[w][cc] - ref);
            total += f[w] * sl[w][cc];
        }
        const int y = first_col + 16 * x + cc;
        if (y < columns) {
            const int64_t r = (((int64_t)set * a.beams + y / per_seq) * a.n + y % per_seq / a.group) * (int64_t)(H * a.group) + h * a.group + y % a.group;
            const int64_t rows = (int64_t)c.num_seqs * a.n * H * a.group;
            const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const int d = 4 * (threadIdx.x & 15) + 64 * k;
                f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WAVES; ++w)
                    if (f[w] != 0.f) v += *reinterpret_cast<const f32x4*>(&so[w][cc][d]) * f[w];
                if (a.splits == 1) {
                    bf16x4 b;
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] = (bf16_t)(v[i] * inv);
                    *reinterpret_cast<bf16x4*>(a.out + r * D + d) = b;
                } else {
                    *reinterpret_cast<f32x4*>(a.part_o + ((int64_t)blockIdx.x * rows + r) * D + d) = v;
                }
            }
            if (a.splits > 1 && (threadIdx.x & 15) == 0) a.part_ml[(int64_t)blockIdx.x * rows + r] = make_float2(top, total);
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
    for (int s = 0; s < splits; ++s) top = fmaxf(top, part_ml[s * rows + r].x);
    const float ref = top > NEG_INF ? top : 0.f;
    float total = 0.f;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        const float2 ml = part_ml[s * rows + r];
        const float f = __builtin_amdgcn_exp2f(ml.x - ref);
        total += f * ml.y;
        if (f != 0.f) v += *reinterpret_cast<const f32x4*>(part_o + (s * rows + r) * D + d) * f;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    bf16x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (bf16_t)(v[i] * inv);
    *reinterpret_cast<bf16x4*>(out + r * D + d) = y;
}

struct Plan {
    int ct, splits, chunks;
    bool own;
};
// Columns enough for four waves of their own: each walks all pages.  Fewer: the waves share them and split the tokens,
// over as many workgroups as fill the card.  By the capacity of the table, not by the lengths, which only the device knows.
Plan plan_of(const asrk_kv_cache* c, int n, int q_heads, int beams) {
    const int64_t columns = (int64_t)beams * n * (q_heads / c->kv_heads);
    Plan p;
    p.own = columns >= 128;
    p.ct = columns > 16 ? 2 : 1;
    const int per = 16 * p.ct * (p.own ? WAVES : 1);
    p.chunks = (int)((columns + per - 1) / per);
    p.splits = 1;
    if (!p.own) {
        const int64_t groups = (int64_t)c->kv_heads * (c->num_seqs / beams) * p.chunks;
        const int64_t want = (2048 + groups - 1) / groups, most = (c->max_pages + WAVES - 1) / WAVES;
        p.splits = (int)(want < most ? want : most);
        if (p.splits > 128) p.splits = 128;
    }
    return p;
}

template <int D, int CT, bool OWN>
void launch(const asrk_kv_cache* c, const AttnArgs& a, int sets, int chunks, hipStream_t st) {
    hipLaunchKernelGGL((kv_attention_kernel<D, CT, OWN>), dim3(a.splits, c->kv_heads, sets * chunks), dim3(256), 0, st, *c, a);
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
    if (layer < 0 || layer >= c->num_layers || seq_ld < 0 || row_ld < 0 || head_ld < 0) return ASRK_ERR_SHAPE;
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
    if (c->head_dim == 64) {
        if (p.own) launch<64, 2, true>(c, a, sets, p.chunks, st);
        else if (p.ct == 2) launch<64, 2, false>(c, a, sets, p.chunks, st);
        else launch<64, 1, false>(c, a, sets, p.chunks, st);
    } else {
        if (p.own) launch<128, 2, true>(c, a, sets, p.chunks, st);
        else if (p.ct == 2) launch<128, 2, false>(c, a, sets, p.chunks, st);
        else launch<128, 1, false>(c, a, sets, p.chunks, st);
    }
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
