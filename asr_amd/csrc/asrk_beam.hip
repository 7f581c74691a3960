// Beam search on the device: the selection over beams and vocabulary, and the reordering of per-beam state.
//
// Selection, for utterance b with K beams over V words, logits x[b,k,:] and running log-probabilities s[b,k]:
//     c(k, v) = s_k + x_kv - log sum_w exp(x_kw)
// and the best n = 2 K of the K V values, ties to the lowest k V + v.  A beam whose score or largest logit is not
// finite, or that holds a NaN, offers -inf throughout.
//
// HBM-bound: every logit is read once, into registers.  Rows are cut into chunks of 8192 so that one utterance already
// gives 7 workgroups per beam at 50 k words; a second, small launch joins the chunks.  (One launch with a last-block
// counter would need that counter cleared, and shared, between calls; two launches need neither.)
#include "asrk_common.h"

namespace {

constexpr int SEL_WAVES = 4;
constexpr int SEL_EPT = 32;                          // logits per lane
constexpr int SEL_CHUNK = SEL_WAVES * 64 * SEL_EPT;  // logits per workgroup
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
    static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    }
};
template <>
struct SelVec<bf16_t> {
    typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r[i] << 16);
            x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
};

// One workgroup per (chunk, row).  Keys are (value, ~index) in 64 bits and hence all different, which bounds the work
// for any input: the n-th largest of the 64 lane maxima of a wave is a lower bound of its n-th largest key, and only
// the n lanes at or above it can hold keys that count, so at most 32 n keys per wave reach LDS (with random logits
// about 1.5 n do).
template <class T>
__global__ __launch_bounds__(256) void beam_chunk_kernel(const T* __restrict__ logits, int64_t ld, int V, int n,
                                                         uint64_t* __restrict__ keys, float2* __restrict__ stats) {
    constexpr int VEC = SelVec<T>::N;
    __shared__ uint64_t cand[SEL_WAVES][SEL_MAX_N * SEL_EPT];
    __shared__ int count[SEL_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.y, chunk = blockIdx.x;
    const T* p = logits + (int64_t)row * ld;
    float x[SEL_EPT];
    int first[SEL_EPT / VEC];
#pragma unroll
    for (int j = 0; j < SEL_EPT / VEC; ++j) {
        const int e = (chunk * SEL_WAVES + wave) * 64 * SEL_EPT + (j * 64 + lane) * VEC;
        first[j] = e;
        if (e + VEC <= V) {
            SelVec<T>::unpack(*reinterpret_cast<const typename SelVec<T>::Raw*>(p + e), x + j * VEC);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[j * VEC + i] = e + i < V ? (float)p[e + i] : NEG_INF;
        }
    }
    float top = NEG_INF;
    bool bad = false;
    uint64_t best = 0;
    auto key = [&](int j, int i) __attribute__((always_inline)) -> uint64_t {
        const int e = first[j] + i;
        return e < V ? ((uint64_t)ord32(x[j * VEC + i]) << 32) | (0xffffffffu - (uint32_t)e) : 0;
    };
#pragma unroll
    for (int j = 0; j < SEL_EPT / VEC; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float& v = x[j * VEC + i];
            bad |= !(v < __builtin_inff());
            v = v + 0.0f;
            top = fmaxf(top, v);
            const uint64_t k = key(j, i);
            best = k > best ? k : best;
        }
    top = wave_max(top);
    float sum = 0.f;
    if (top > NEG_INF) {
#pragma unroll
        for (int i = 0; i < SEL_EPT; ++i) sum += __builtin_amdgcn_exp2f((x[i] - top) * 1.4426950408889634f);
    }
    sum = wave_sum(sum);
    bad = __any(bad);
    if (lane == 0)
        stats[((int64_t)row * gridDim.x + chunk) * SEL_WAVES + wave] = make_float2(bad ? __builtin_inff() : top, sum);

    // the wave's threshold: the lane maximum of rank n - 1
    int rank = 0;
    const uint32_t bh = (uint32_t)(best >> 32), bl = (uint32_t)best;
#pragma unroll 8
    for (int l = 0; l < 64; ++l) {
        const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(bh, l) << 32) | (uint32_t)__builtin_amdgcn_readlane(bl, l);
        rank += o > best ? 1 : 0;
    }
    const uint64_t at = __ballot(rank == n - 1 && best != 0);
    uint64_t tau = 1;  // fewer than n lanes hold anything: all of it counts
    if (at) {
        const int l = __builtin_ctzll(at);
        tau = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(bh, l) << 32) | (uint32_t)__builtin_amdgcn_readlane(bl, l);
    }
    int c = 0;
    if (__any(best >= tau)) {
#pragma unroll
        for (int j = 0; j < SEL_EPT / VEC; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint64_t k = key(j, i);
                const uint64_t m = __ballot(k >= tau);
                if (m) {
                    if (k >= tau) cand[wave][c + __popcll(m & ((1ull << lane) - 1))] = k;
                    c += __popcll(m);
                }
            }
    }
    if (lane == 0) count[wave] = c;
    __syncthreads();
    uint64_t* out = keys + ((int64_t)row * gridDim.x + chunk) * n;
    int total = 0;
#pragma unroll
    for (int w = 0; w < SEL_WAVES; ++w) total += count[w];
    for (int r = total + (int)threadIdx.x; r < n; r += 256) out[r] = 0;
    for (int w = 0; w < SEL_WAVES; ++w)
        for (int t = threadIdx.x; t < count[w]; t += 256) {
            const uint64_t mine = cand[w][t];
            int r = 0;
            for (int w2 = 0; w2 < SEL_WAVES; ++w2)
                for (int u = 0; u < count[w2]; ++u) r += cand[w2][u] > mine ? 1 : 0;
            if (r < n) out[r] = mine;
        }
}

struct Pick {
    double v;
    uint32_t at;
};
__device__ __forceinline__ bool ahead(const Pick& a, const Pick& b) { return a.v > b.v || (a.v == b.v && a.at < b.at); }

// One workgroup per utterance: the row sums in 64 bits, then the best n of the chunks' sorted lists.  Values are
// compared in 64 bits, where different logits of a beam stay different (and equal ones equal); the n-th best list head
// bounds the n-th best value from below, so at most n lists of at most n keys are looked at.
__global__ __launch_bounds__(256) void beam_join_kernel(const uint64_t* __restrict__ keys, const float2* __restrict__ stats,
                                                        const float* __restrict__ scores, int K, int V, int chunks, int n,
                                                        int64_t eos, float* __restrict__ out_scores,
                                                        int64_t* __restrict__ out_tokens, int64_t* __restrict__ out_parents,
                                                        float* __restrict__ cand_scores, int64_t* __restrict__ cand_tokens,
                                                        int64_t* __restrict__ cand_parents) {
    __shared__ double lse[SEL_MAX_BEAMS];
    __shared__ double score[SEL_MAX_BEAMS];
    __shared__ int alive[SEL_MAX_BEAMS];
    __shared__ double head_v[SEL_MAX_LISTS];
    __shared__ uint32_t head_at[SEL_MAX_LISTS];
    __shared__ double cand_v[SEL_MAX_N * SEL_MAX_N];
    __shared__ uint32_t cand_at[SEL_MAX_N * SEL_MAX_N];
    __shared__ Pick tau;
    __shared__ int n_cand;
    __shared__ double best_v[SEL_MAX_N];
    __shared__ uint32_t best_at[SEL_MAX_N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.x;
    if (threadIdx.x == 0) {
        n_cand = 0;
        tau = Pick{-__builtin_inf(), 0xffffffffu};  // everything is ahead of it
    }
    for (int k = wave; k < K; k += 4) {
        const float2* st = stats + ((int64_t)b * K + k) * chunks * SEL_WAVES;
        float top = NEG_INF;
        for (int i = lane; i < chunks * SEL_WAVES; i += 64) top = fmaxf(top, st[i].x);
        top = wave_max(top);
        double sum = 0.0;
        const bool ok = top > NEG_INF && top < __builtin_inff();
        if (ok)
            for (int i = lane; i < chunks * SEL_WAVES; i += 64)
                if (st[i].x > NEG_INF) sum += (double)st[i].y * exp((double)st[i].x - (double)top);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) {
            const float s = scores[(int64_t)b * K + k];
            alive[k] = ok && s > NEG_INF && s < __builtin_inff();
            lse[k] = ok ? (double)top + log(sum) : 0.0;
            score[k] = (double)s;
        }
    }
    __syncthreads();
    const int lists = K * chunks;
    // entry j of list l; false: none
    auto entry = [&](int l, int j, Pick& p) -> bool {
        const int k = l / chunks, c = l - k * chunks;
        if (!alive[k]) {  // a dead beam: its words in order
            p = Pick{-__builtin_inf(), (uint32_t)(k * V + j)};
            return c == 0 && j < V;
        }
        const uint64_t key = keys[(((int64_t)b * K + k) * chunks + c) * n + j];
        p = Pick{score[k] + ((double)unord32((uint32_t)(key >> 32)) - lse[k]), (uint32_t)(k * V) + (0xffffffffu - (uint32_t)key)};
        return key != 0;
    };
    for (int l = threadIdx.x; l < lists; l += 256) {
        Pick p;
        const bool any = entry(l, 0, p);
        head_v[l] = any ? p.v : __builtin_nan("");
        head_at[l] = any ? p.at : 0xffffffffu;
    }
    __syncthreads();
    for (int l = threadIdx.x; l < lists; l += 256) {
        const Pick mine{head_v[l], head_at[l]};
        if (mine.v != mine.v) continue;
        int r = 0;
        for (int u = 0; u < lists; ++u) r += ahead(Pick{head_v[u], head_at[u]}, mine) ? 1 : 0;  // NaN is ahead of nothing
        if (r == n - 1) tau = mine;
    }
    __syncthreads();
    const Pick least = tau;
    for (int l = threadIdx.x; l < lists; l += 256) {
        Pick p{head_v[l], head_at[l]};
        if (p.v != p.v) continue;
        for (int j = 0; j < n; ++j) {
            if (j > 0 && !entry(l, j, p)) break;
            if (ahead(least, p)) break;  // lists are sorted
            const int at = atomicAdd(&n_cand, 1);
            cand_v[at] = p.v;
            cand_at[at] = p.at;
        }
    }
    __syncthreads();
    const int c = n_cand;
    for (int t = threadIdx.x; t < c; t += 256) {
        const Pick mine{cand_v[t], cand_at[t]};
        int r = 0;
        for (int u = 0; u < c; ++u) r += ahead(Pick{cand_v[u], cand_at[u]}, mine) ? 1 : 0;
        if (r < n) {
            best_v[r] = mine.v;
            best_at[r] = mine.at;
        }
    }
    __syncthreads();
    if (wave == 0) {  // n <= 32 lanes
        const bool in = lane < n;
        const uint32_t at = in ? best_at[lane] : 0;
        const int64_t parent = at / (uint32_t)V, token = at % (uint32_t)V;
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

int sel_chunks(int V) { return (int)(((int64_t)V + SEL_CHUNK - 1) / SEL_CHUNK); }

}  // namespace

extern "C" size_t asrk_beam_select_workspace_bytes(int B, int K, int V) {
    if (B <= 0 || K <= 0 || K > SEL_MAX_BEAMS || V < 2) return 0;
    return (size_t)B * K * sel_chunks(V) * (2 * K * sizeof(uint64_t) + SEL_WAVES * sizeof(float2));
}

extern "C" int asrk_beam_select(const void* logits, int dtype, int64_t ld, const float* scores, int B, int K, int V, int64_t eos,
                                float* out_scores, int64_t* out_tokens, int64_t* out_parents, float* cand_scores,
                                int64_t* cand_tokens, int64_t* cand_parents, void* ws, size_t ws_bytes, void* stream) {
    if (!logits || !scores || !out_scores || !out_tokens || !out_parents || !cand_scores || !cand_tokens || !cand_parents || !ws)
        return ASRK_ERR_NULL;
    if (dtype != ASRK_F32 && dtype != ASRK_BF16) return ASRK_ERR_UNSUPPORTED;
    if (B <= 0 || K <= 0 || K > SEL_MAX_BEAMS || V < 2 || ld < V || (int64_t)B * K > 65535 || (int64_t)K * V > 0x7fffffff)
        return ASRK_ERR_SHAPE;
    const int chunks = sel_chunks(V);
    if (K * chunks > SEL_MAX_LISTS) return ASRK_ERR_SHAPE;
    if ((uintptr_t)logits % (dtype == ASRK_F32 ? 4 : 2)) return ASRK_ERR_ALIGN;
    if ((uintptr_t)ws & 15) return ASRK_ERR_ALIGN;
    if (ws_bytes < asrk_beam_select_workspace_bytes(B, K, V)) return ASRK_ERR_WORKSPACE;
    uint64_t* keys = (uint64_t*)ws;
    float2* stats = (float2*)(keys + (size_t)B * K * chunks * 2 * K);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ASRK_F32)
        hipLaunchKernelGGL(beam_chunk_kernel<float>, dim3(chunks, B * K), dim3(256), 0, st, (const float*)logits, ld, V, 2 * K, keys,
                           stats);
    else
        hipLaunchKernelGGL(beam_chunk_kernel<bf16_t>, dim3(chunks, B * K), dim3(256), 0, st, (const bf16_t*)logits, ld, V, 2 * K,
                           keys, stats);
    hipLaunchKernelGGL(beam_join_kernel, dim3(B), dim3(256), 0, st, keys, stats, scores, K, V, chunks, 2 * K, eos, out_scores,
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
