// Beam search on the device: the selection over beams and vocabulary, and the reordering of per-beam state.
//
// Selection, for utterance b with K beams over V words, logits x[b,k,:] and running log-probabilities s[b,k]:
//     c(k, v) = s_k + x_kv - log sum_w exp(x_kw)
// and the best n = 2 K of the K V values, ties to the lowest k V + v.  A beam whose score or largest logit is not
// finite, or that holds a NaN, offers -inf throughout.
//
// HBM-bound where it is large (32 x 8 beams, 128001 fp32 words, 131 MB: chunk kernel 25.9 us = 5.1 TB/s, join 8.6; 64 x 5,
// 51865 bf16 words, 33 MB: 13.9 and 5.7, bound by instructions and latency): every logit is read once, into registers.  Rows
// are cut into chunks of 8192 so that one utterance already
// gives 7 workgroups per beam at 50 k words; a second, small launch joins the chunks.  (One launch with a last-block
// counter would need that counter cleared, and shared, between calls; two launches need neither.)
#include "asrk_common.h"

namespace {

constexpr int SEL_WAVES = 4;
constexpr int SEL_CHUNK = 8192;  // logits per workgroup: 32 per lane, or twice that
constexpr int SEL_MAX_BEAMS = 16;
constexpr int SEL_MAX_N = 2 * SEL_MAX_BEAMS;
constexpr int SEL_MAX_LISTS = 2048;
constexpr float NEG_INF = -__builtin_inff();

// order-preserving map of a float to an unsigned integer (no NaN; -0 was made +0)
__device__ __forceinline__ uint32_t ord32(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord32(uint32_t o) {
    return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// Rows of an odd vocabulary start anywhere: the 16-byte loads are aligned to the value only, so that a row is cut into
// the same pieces, and sums to the same bits, wherever it lies (equal beams must stay equal).
template <class T>
struct SelVec;
template <>
struct SelVec<float> {
    typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int N = 4;
    static __device__ __forceinline__ u32x4 place(float v, int i) {
        const uint32_t w = __float_as_uint(v);
        return u32x4{i == 0 ? w : 0, i == 1 ? w : 0, i == 2 ? w : 0, i == 3 ? w : 0};
    }
    static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    }
};
template <>
struct SelVec<bf16_t> {
    typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
    static constexpr int N = 8;
    static __device__ __forceinline__ u32x4 place(bf16_t v, int i) {
        const uint32_t w = (__float_as_uint((float)v) >> 16) << (16 * (i & 1));
        return u32x4{i / 2 == 0 ? w : 0, i / 2 == 1 ? w : 0, i / 2 == 2 ? w : 0, i / 2 == 3 ? w : 0};
    }
    static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r[i] << 16);
            x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
};

// Maximum and sum over a wave: shifts within rows of 16, then rows broadcast to later ones.
template <int CONTROL, int ROWS>
__device__ __forceinline__ float from_lane(float v, float none) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(none), __float_as_uint(v), CONTROL, ROWS, 0xf, false));
}
template <class F>
__device__ __forceinline__ float over_wave(float v, float none, F&& f) {
    v = f(v, from_lane<0x111, 0xf>(v, none));
    v = f(v, from_lane<0x112, 0xf>(v, none));
    v = f(v, from_lane<0x114, 0xf>(v, none));
    v = f(v, from_lane<0x118, 0xf>(v, none));
    v = f(v, from_lane<0x142, 0xa>(v, none));
    v = f(v, from_lane<0x143, 0xc>(v, none));
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
__device__ __forceinline__ float sel_max(float v) { return over_wave(v, NEG_INF, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float sel_sum(float v) { return over_wave(v, 0.f, [](float a, float b) { return a + b; }); }

constexpr int sel_lanes(int n) { return n + 8; }  // lanes of a workgroup whose values may be candidates

// One workgroup per (chunk, row).  A threshold with at least n of the 256 lane maxima at or above it is a lower bound of
// the chunk's n-th best value, and only those lanes can hold values that count.  Bisection finds one with n .. n + 8 such
// lanes in a few steps, a compare and a bit count per wave's worth of lanes; every wave does it for itself on all 256.
// Where equal values leave no such threshold it falls back to ranking the lane maxima by (value, ~word), which are all
// different.  Either way at most sel_lanes(n) lanes of 32 (64) keys reach LDS, for any input (with random logits about n + 6
// keys do).
template <class T, int SEL_EPT>  // logits per lane
__global__ __launch_bounds__(256) void beam_chunk_kernel(const T* __restrict__ logits, int64_t ld, int V, int n,
                                                         uint64_t* __restrict__ keys, float2* __restrict__ stats) {
    constexpr int VEC = SelVec<T>::N;
    extern __shared__ uint64_t cand[];  // [sel_lanes(n) * SEL_EPT]
    __shared__ __attribute__((aligned(16))) uint32_t bests[256];
    __shared__ uint32_t firsts[256];
    __shared__ int count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.y, chunk = blockIdx.x;
    const T* p = logits + (int64_t)row * ld;
    const int e0 = (chunk * SEL_WAVES + wave) * 64 * SEL_EPT + lane * VEC;  // word of slot 0
    // A piece that passes the row's end is taken so that it ends there; what it then has in common with the piece in front, and
    // all of the pieces behind, is masked.
    const int last = V - VEC;
    auto nominal = [&](int s) __attribute__((always_inline)) { return e0 + s / VEC * 64 * VEC; };
    auto begin = [&](int s) __attribute__((always_inline)) { return nominal(s) < last ? nominal(s) : last; };
    auto word = [&](int s) __attribute__((always_inline)) { return begin(s) + s % VEC; };  // ascending
    auto real = [&](int s) __attribute__((always_inline)) { return s % VEC >= nominal(s) - begin(s); };
    float x[SEL_EPT];
    const int first_word = __builtin_amdgcn_readfirstlane(e0);
    if (first_word >= V) {
#pragma unroll
        for (int s = 0; s < SEL_EPT; ++s) x[s] = NEG_INF;
    } else {
        u32x4 raw[SEL_EPT / VEC];
        if (V >= VEC) {
#pragma unroll
            for (int j = 0; j < SEL_EPT / VEC; ++j) raw[j] = *reinterpret_cast<const typename SelVec<T>::Raw*>(p + begin(j * VEC));
        } else {
#pragma unroll
            for (int j = 0; j < SEL_EPT / VEC; ++j) raw[j] = u32x4{0, 0, 0, 0};
            for (int i = 0; i < V; ++i) raw[0] |= SelVec<T>::place(p[i], i - last);
        }
#pragma unroll
        for (int j = 0; j < SEL_EPT / VEC; ++j) SelVec<T>::unpack(raw[j], x + j * VEC);
        if (first_word + 64 * SEL_EPT > V) {
            asm volatile("");  // a branch: masks cost whole waves as much as the maximum does
#pragma unroll
            for (int s = 0; s < SEL_EPT; ++s) x[s] = real(s) ? x[s] : NEG_INF;
        }
    }
    float best = NEG_INF;
#pragma unroll
    for (int s = 0; s < SEL_EPT; ++s) best = fmaxf(best, x[s]);
    // the lane maxima of all four waves, lane l of wave w at 4 l + w; 0: no word at all
    bests[lane * 4 + wave] = e0 < V ? ord32(best + 0.0f) : 0;  // -0 counts as 0
    if (threadIdx.x == 0) count = 0;
    const float top = sel_max(best);
    const float ref = top > NEG_INF ? top : 0.f;
    float sum = 0.f;  // NaN if one of the logits is
#pragma unroll
    for (int s = 0; s < SEL_EPT; ++s) sum += __builtin_amdgcn_exp2f((x[s] - ref) * 1.4426950408889634f);
    sum = sel_sum(sum);
    if (lane == 0)
        stats[((int64_t)row * gridDim.x + chunk) * SEL_WAVES + wave] = make_float2(sum == sum ? top : __builtin_inff(), sum);
    __syncthreads();

    constexpr uint32_t LOWEST = 0x007fffffu;  // -inf
    const u32x4 mine = *reinterpret_cast<const u32x4*>(bests + lane * 4);
    auto at_least = [&](uint32_t t) __attribute__((always_inline)) {
        int c = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) c += __popcll(__ballot(mine[w] >= t));
        return c;
    };
    uint32_t tau = LOWEST, tau_low = 0;  // n lanes or fewer hold anything: all of it counts
    if (at_least(1) > n) {
        uint32_t lo = LOWEST, hi = 0xff800001u;  // at or above lo: too many; hi: too few (above +inf)
        bool found = false;
        {  // most lane maxima lie within a few units below the largest
            float m = sel_max(fmaxf(fmaxf(unord32(mine[0] ? mine[0] : LOWEST), unord32(mine[1] ? mine[1] : LOWEST)),
                                     fmaxf(unord32(mine[2] ? mine[2] : LOWEST), unord32(mine[3] ? mine[3] : LOWEST))));
            hi = __builtin_amdgcn_readfirstlane(ord32(m)) + 1;
        }
        while (!found && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int c = at_least(mid);
            found = c >= n && c <= sel_lanes(n);
            if (found) tau = mid;
            else if (c < n) hi = mid;
            else lo = mid;
        }
        if (!found) {  // the n-th lane by (value, ~word)
            uint32_t first = 0;
#pragma unroll
            for (int s = SEL_EPT - 1; s >= 0; --s) first = x[s] == best && real(s) ? 0xffffffffu - (uint32_t)word(s) : first;
            firsts[lane * 4 + wave] = first;
            __syncthreads();  // every wave is here: they all look at the same 256 values
            for (int w = 0; w < 4; ++w) {
                const uint64_t key = ((uint64_t)bests[lane * 4 + w] << 32) | firsts[lane * 4 + w];
                int rank = 0;
#pragma unroll 4
                for (int l = 0; l < 256; ++l) rank += (((uint64_t)bests[l] << 32) | firsts[l]) > key ? 1 : 0;
                const uint64_t m = __ballot(rank == n - 1 && key >> 32);
                if (m) {
                    tau = __builtin_amdgcn_readlane((uint32_t)(key >> 32), __builtin_ctzll(m));
                    tau_low = __builtin_amdgcn_readlane((uint32_t)key, __builtin_ctzll(m));
                }
            }
        }
    }
    const float least = unord32(tau);
    if (__any(best >= least)) {
#pragma unroll
        for (int s = 0; s < SEL_EPT; ++s) {
            if (!__any(x[s] >= least)) continue;
            const uint32_t high = ord32(x[s] + 0.0f), low = 0xffffffffu - (uint32_t)word(s);
            if (x[s] >= least && real(s) && (high > tau || low >= tau_low)) cand[atomicAdd(&count, 1)] = ((uint64_t)high << 32) | low;
        }
    }
    __syncthreads();
    uint64_t* out = keys + ((int64_t)row * gridDim.x + chunk) * n;
    const int total = count;
    for (int r = total + (int)threadIdx.x; r < n; r += 256) out[r] = 0;
    const int part = threadIdx.x & 3;  // four threads per key, each against a quarter of them
    for (int t = threadIdx.x >> 2; t < (total + 63) / 64 * 64; t += 64) {
        const uint64_t key = t < total ? cand[t] : 0;
        int r = 0;
        for (int u0 = part; u0 < total; u0 += 16)
#pragma unroll
            for (int u = u0; u < u0 + 16; u += 4) r += (u < total) & (cand[u < total ? u : 0] > key);
        r += __shfl_xor(r, 1, 64);
        r += __shfl_xor(r, 2, 64);
        if (part == 0 && t < total && r < n) out[r] = key;
    }
}

// A value, and what decides between equal ones.  Of two words of a beam the one with the larger logit is ahead, also where 64 bits
// cannot tell score + (logit - lse) apart (fp32 logits of 1e-18, a score of -1e30); else the lower beam, then the lower word.
// This is the order in which a chunk's list is sorted.
struct Pick {
    double v;
    uint64_t tie;  // beam, the logit's place from above, word
};
constexpr int WORD_BITS = 25;  // SEL_MAX_LISTS chunks of twice SEL_CHUNK words at most
static_assert((int64_t)SEL_MAX_LISTS * 2 * SEL_CHUNK <= 1 << WORD_BITS && SEL_MAX_BEAMS <= 1 << (64 - 32 - WORD_BITS), "does not fit a tie");
__device__ __forceinline__ uint64_t tie_of(int k, uint32_t ord, uint32_t word) {
    return (uint64_t)k << (32 + WORD_BITS) | (uint64_t)(0xffffffffu - ord) << WORD_BITS | word;
}
__device__ __forceinline__ bool ahead(const Pick& a, const Pick& b) { return (a.v > b.v) | ((a.v == b.v) & (a.tie < b.tie)); }

// One workgroup per utterance: the row sums in 64 bits, then the best n of the chunks' sorted lists.  Values are compared in 64
// bits; the n-th best list head bounds the n-th best value from below, so at most n lists of at most n keys are candidates.
// Bound by its chain of dependent steps: everything it may need is loaded first (a load is about a microsecond, the arithmetic
// is less).
constexpr int JOIN_T = 512;
constexpr int JOIN_HELD = 4;  // keys per thread that are loaded ahead: all of them up to 2048
__device__ __forceinline__ int over(int x, float inverse) { return (int)(((float)x + 0.5f) * inverse); }  // exact: x < 2^16, divisors up to 2048
template <int CONTROL, int ROWS>
__device__ __forceinline__ double from_lane(double v) {  // 0 where there is none
    const uint64_t b = __double_as_longlong(v);
    const uint32_t low = __builtin_amdgcn_update_dpp(0, (uint32_t)b, CONTROL, ROWS, 0xf, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), CONTROL, ROWS, 0xf, false);
    return __longlong_as_double((int64_t)(((uint64_t)high << 32) | low));
}
__global__ __launch_bounds__(JOIN_T) void beam_join_kernel(const uint64_t* __restrict__ keys, const float2* __restrict__ stats,
                                                           const float* __restrict__ scores, int K, int V, int chunks, int n, float chunks_inv, float n_inv,
                                                           int64_t eos, float* __restrict__ out_scores,
                                                           int64_t* __restrict__ out_tokens, int64_t* __restrict__ out_parents,
                                                           float* __restrict__ cand_scores, int64_t* __restrict__ cand_tokens,
                                                           int64_t* __restrict__ cand_parents) {
    __shared__ uint64_t ahead_keys[JOIN_HELD * JOIN_T];
    __shared__ double lse[SEL_MAX_BEAMS];
    __shared__ double score[SEL_MAX_BEAMS];
    __shared__ int alive[SEL_MAX_BEAMS];
    __shared__ double head_v[SEL_MAX_LISTS];
    __shared__ uint64_t head_tie[SEL_MAX_LISTS];
    __shared__ double cand_v[SEL_MAX_N * SEL_MAX_N];
    __shared__ uint64_t cand_tie[SEL_MAX_N * SEL_MAX_N];
    __shared__ Pick tau;
    __shared__ int n_cand;
    __shared__ double best_v[SEL_MAX_N];
    __shared__ uint64_t best_tie[SEL_MAX_N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.x;
    const int lists = K * chunks, all = lists * n;
    const uint64_t* mine = keys + (int64_t)b * all;
    uint64_t held[JOIN_HELD];
#pragma unroll
    for (int q = 0; q < JOIN_HELD; ++q) {
        const int i = q * JOIN_T + threadIdx.x;
        held[q] = i < all ? mine[i] : 0;
    }
    if (threadIdx.x == 0) {
        n_cand = 0;
        tau = Pick{-__builtin_inf(), ~0ull};  // everything is ahead of it
    }
    for (int k = wave; k < K; k += JOIN_T / 64) {
        const float2* st = stats + ((int64_t)b * K + k) * chunks * SEL_WAVES;
        const float s = scores[(int64_t)b * K + k];
        const float2 first = lane < chunks * SEL_WAVES ? st[lane] : make_float2(NEG_INF, 0.f);
        float top = first.x;
        for (int i = lane + 64; i < chunks * SEL_WAVES; i += 64) top = fmaxf(top, st[i].x);
        top = sel_max(top);
        const bool ok = top > NEG_INF && top < __builtin_inff();
        double sum = 0.0;
        if (ok)
            for (int i = lane; i < chunks * SEL_WAVES; i += 64) {
                const float2 one = i == lane ? first : st[i];
                if (one.x > NEG_INF) sum += (double)one.y * exp((double)one.x - (double)top);
            }
        sum += from_lane<0x111, 0xf>(sum);
        sum += from_lane<0x112, 0xf>(sum);
        sum += from_lane<0x114, 0xf>(sum);
        sum += from_lane<0x118, 0xf>(sum);
        sum += from_lane<0x142, 0xa>(sum);
        sum += from_lane<0x143, 0xc>(sum);
        if (lane == 63) {
            alive[k] = ok && s > NEG_INF && s < __builtin_inff();
            lse[k] = ok ? (double)top + log(sum) : 0.0;
            score[k] = (double)s;
        }
    }
#pragma unroll
    for (int q = 0; q < JOIN_HELD; ++q) ahead_keys[q * JOIN_T + threadIdx.x] = held[q];
    __syncthreads();
    // entry j of list l, whose key is `key`; false: none
    auto entry = [&](int l, int j, uint64_t key, Pick& p) -> bool {
        const int k = over(l, chunks_inv);
        if (!alive[k]) {  // a dead beam: its words in order
            p = Pick{-__builtin_inf(), tie_of(k, 0, j)};
            return l == k * chunks && j < V;
        }
        p = Pick{score[k] + ((double)unord32((uint32_t)(key >> 32)) - lse[k]), tie_of(k, (uint32_t)(key >> 32), 0xffffffffu - (uint32_t)key)};
        return key != 0;
    };
    auto each = [&](auto&& f) __attribute__((always_inline)) {  // f(list, place in it, key)
        for (int i = threadIdx.x; i < all; i += JOIN_T) {
            const int l = over(i, n_inv);
            f(l, i - l * n, i < JOIN_HELD * JOIN_T ? ahead_keys[i] : mine[i]);
        }
    };
    each([&](int l, int j, uint64_t key) {
        if (j) return;
        Pick p;
        const bool any = entry(l, 0, key, p);
        head_v[l] = any ? p.v : __builtin_nan("");
        head_tie[l] = any ? p.tie : ~0ull;
    });
    __syncthreads();
    const int part = threadIdx.x & 3;  // four threads per head, and per candidate, each against a quarter of the others
    for (int l = threadIdx.x >> 2; l < lists; l += JOIN_T / 4) {
        const Pick p{head_v[l], head_tie[l]};
        int r = 0;
        for (int u0 = part; u0 < lists; u0 += 16)
#pragma unroll
            for (int u = u0; u < u0 + 16; u += 4) r += (u < lists) & ahead(Pick{head_v[u], head_tie[u]}, p);  // NaN is ahead of nothing
        r += __shfl_xor(r, 1, 64);
        r += __shfl_xor(r, 2, 64);
        if (part == 0 && r == n - 1 && p.v == p.v) tau = p;
    }
    __syncthreads();
    const Pick least = tau;
    each([&](int l, int j, uint64_t key) {
        if (head_v[l] != head_v[l] || ahead(least, Pick{head_v[l], head_tie[l]})) return;
        Pick p;
        if (!entry(l, j, key, p) || ahead(least, p)) return;
        const int at = atomicAdd(&n_cand, 1);
        cand_v[at] = p.v;
        cand_tie[at] = p.tie;
    });
    __syncthreads();
    const int c = n_cand;
    for (int t = threadIdx.x >> 2; t < c; t += JOIN_T / 4) {
        const Pick p{cand_v[t], cand_tie[t]};
        int r = 0;
        for (int u0 = part; u0 < c; u0 += 16)
#pragma unroll
            for (int u = u0; u < u0 + 16; u += 4) r += (u < c) & ahead(Pick{cand_v[u], cand_tie[u]}, p);
        r += __shfl_xor(r, 1, 64);
        r += __shfl_xor(r, 2, 64);
        if (part == 0 && r < n) {
            best_v[r] = p.v;
            best_tie[r] = p.tie;
        }
    }
    __syncthreads();
    if (wave == 0) {  // n <= 32 lanes
        const bool in = lane < n;
        const uint64_t tie = in ? best_tie[lane] : 0;
        const int64_t parent = tie >> (32 + WORD_BITS), token = tie & ((1 << WORD_BITS) - 1);
        const float v = in ? (float)best_v[lane] : 0.f;
        if (in) {
            cand_scores[(int64_t)b * n + lane] = v;
            cand_tokens[(int64_t)b * n + lane] = token;
            cand_parents[(int64_t)b * n + lane] = parent;
        }
        const bool go = in && token != eos;
        const uint64_t m = __ballot(go);
        const int r = __popcll(m & ((1ull << lane) - 1));
        if (go && r < K) {
            out_scores[(int64_t)b * K + r] = v;
            out_tokens[(int64_t)b * K + r] = token;
            out_parents[(int64_t)b * K + r] = parent;
        }
    }
}

// out[b][k] = in[b][parents[b][k]]: rows of `units` elements of T, the grid's y is the row.
template <class T>
__global__ __launch_bounds__(256) void reorder_rows_kernel(const T* __restrict__ in, const int64_t* __restrict__ parents, int K,
                                                           int64_t units, T* __restrict__ out) {
    const int64_t row = blockIdx.y;
    const int64_t b = row / K;
    int64_t p = parents[row];
    p = p < 0 || p >= K ? row - b * K : p;  // not a beam: the row stays
    const T* src = in + (b * K + p) * units;
    T* dst = out + row * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < units; i += (int64_t)gridDim.x * 256) dst[i] = src[i];
}

int sel_chunks(int V, int chunk) { return (int)(((int64_t)V + chunk - 1) / chunk); }

// bf16 rows are bound by instructions, and what a workgroup does besides its logits halves with twice as many of them; so
// where there are workgroups for more than one round of the card (8 on each of 256 CUs), it takes them: 64 x 5 rows of
// 51865 words 17.1 -> 14.4 us.  fp32 rows are bound by memory: 32 x 8 rows of 128001 words 27.3 -> 28.8 us, not taken.
int sel_chunk(int dtype, int64_t rows, int V) {
    return dtype == ASRK_BF16 && rows * sel_chunks(V, SEL_CHUNK) > 2048 ? 2 * SEL_CHUNK : SEL_CHUNK;
}

}  // namespace

extern "C" size_t asrk_beam_select_workspace_bytes(int B, int K, int V) {
    if (B <= 0 || K <= 0 || K > SEL_MAX_BEAMS || V < 2) return 0;
    return (size_t)B * K * sel_chunks(V, SEL_CHUNK) * (2 * K * sizeof(uint64_t) + SEL_WAVES * sizeof(float2));
}

extern "C" int asrk_beam_select(const void* logits, int dtype, int64_t ld, const float* scores, int B, int K, int V, int64_t eos,
                                float* out_scores, int64_t* out_tokens, int64_t* out_parents, float* cand_scores,
                                int64_t* cand_tokens, int64_t* cand_parents, void* ws, size_t ws_bytes, void* stream) {
    if (!logits || !scores || !out_scores || !out_tokens || !out_parents || !cand_scores || !cand_tokens || !cand_parents || !ws)
        return ASRK_ERR_NULL;
    if (dtype != ASRK_F32 && dtype != ASRK_BF16) return ASRK_ERR_UNSUPPORTED;
    if (B <= 0 || K <= 0 || K > SEL_MAX_BEAMS || V < 2 || ld < V || (int64_t)B * K > 65535 || (int64_t)K * V > 0x7fffffff)
        return ASRK_ERR_SHAPE;
    const int chunk = sel_chunk(dtype, (int64_t)B * K, V), chunks = sel_chunks(V, chunk);
    if (K * chunks > SEL_MAX_LISTS) return ASRK_ERR_SHAPE;
    if ((uintptr_t)logits % (dtype == ASRK_F32 ? 4 : 2)) return ASRK_ERR_ALIGN;
    if ((uintptr_t)ws & 15) return ASRK_ERR_ALIGN;
    if (ws_bytes < asrk_beam_select_workspace_bytes(B, K, V)) return ASRK_ERR_WORKSPACE;
    uint64_t* keys = (uint64_t*)ws;
    float2* stats = (float2*)(keys + (size_t)B * K * chunks * 2 * K);
    hipStream_t st = (hipStream_t)stream;
    const size_t lds = (size_t)sel_lanes(2 * K) * (chunk / 256) * sizeof(uint64_t);  // 20 KiB at most
    const dim3 grid(chunks, B * K);
    if (dtype == ASRK_F32)
        hipLaunchKernelGGL((beam_chunk_kernel<float, 32>), grid, dim3(256), lds, st, (const float*)logits, ld, V, 2 * K, keys, stats);
    else if (chunk == SEL_CHUNK)
        hipLaunchKernelGGL((beam_chunk_kernel<bf16_t, 32>), grid, dim3(256), lds, st, (const bf16_t*)logits, ld, V, 2 * K, keys, stats);
    else
        hipLaunchKernelGGL((beam_chunk_kernel<bf16_t, 64>), grid, dim3(256), lds, st, (const bf16_t*)logits, ld, V, 2 * K, keys, stats);
    hipLaunchKernelGGL(beam_join_kernel, dim3(B), dim3(JOIN_T), 0, st, keys, stats, scores, K, V, chunks, 2 * K, 1.f / chunks, 0.5f / K, eos, out_scores,
                       out_tokens, out_parents, cand_scores, cand_tokens, cand_parents);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}

extern "C" int asrk_reorder_rows(const void* in, const int64_t* parents, int B, int K, int64_t row_bytes, void* out, void* stream) {
    if (!in || !parents || !out) return ASRK_ERR_NULL;
    if (B <= 0 || K <= 0 || row_bytes <= 0 || (int64_t)B * K > 65535) return ASRK_ERR_SHAPE;
    const int64_t rows = (int64_t)B * K;
    const bool wide = !(((uintptr_t)in | (uintptr_t)out | (uintptr_t)row_bytes) & 15);
    const int64_t units = wide ? row_bytes / 16 : row_bytes;
    const int64_t want = (units + 255) / 256, most = (16384 + rows - 1) / rows;  // enough blocks to fill the card, then loops
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)rows);
    hipStream_t st = (hipStream_t)stream;
    if (wide)
        hipLaunchKernelGGL(reorder_rows_kernel<u32x4>, grid, dim3(256), 0, st, (const u32x4*)in, parents, K, units, (u32x4*)out);
    else
        hipLaunchKernelGGL(reorder_rows_kernel<uint8_t>, grid, dim3(256), 0, st, (const uint8_t*)in, parents, K, units, (uint8_t*)out);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}
