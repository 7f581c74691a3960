// The paged 8-bit key/value cache: its pages, and how tokens get in and out.
//
// A page holds 64 tokens of one key/value head, keys [64][D] and values transposed [D][64] (what the attention's matrix
// instructions read without a shuffle), in e4m3 with one power-of-two scale each: x = q 2^e.  A power of two makes the
// scaling itself exact: the only rounding is the one to e4m3's 3 bits (half a step, 2^-4 relative), every value held is
// also a bf16 value, and when a later token raises the page's exponent the older ones are re-rounded exactly, but for
// those that become subnormal.  e is the smallest integer with max|x| <= 448 2^e, clamped to [-64, 119]: at 119 the
// largest value is 1.75 2^127, still a finite bf16 (larger inputs saturate there); below -64 everything is zero.
// NaN and infinities are stored as NaN and take no part in the scale.
//
// Pages belong to sequences through `table`, with a count of holders per page (`refs`, 0 = free).  All of it lives on
// the device, so that a decoding step needs no host round trip and can be captured into a graph.
#include "asrk_kvcache.h"

namespace {

constexpr int MANAGE_T = 1024;  // threads of the one-workgroup kernels

// Inclusive sums over a wave, or over its first 16 lanes (ROW): shifts within rows of 16, then rows broadcast to later ones.
template <bool ROW>
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    if (!ROW) {
        x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
        x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    }
    return x;
}
__device__ __forceinline__ int block_scan_exclusive(int v, int* lds, int& total) {  // MANAGE_T threads, 16 waves
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = wave_scan<false>(v);
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    const int w = lds[lane & 15], upto = wave_scan<true>(w);
    total = __builtin_amdgcn_readlane(upto, 15);
    const int before = __builtin_amdgcn_readlane(upto, wave) - __builtin_amdgcn_readlane(w, wave);
    __syncthreads();
    return before + x - v;
}

// The page that token `len` of a sequence goes into, if the sequence has it already; -1: a fresh one.
__device__ __forceinline__ int open_page(const asrk_kv_cache& c, int64_t slot, int len) {
    if (len % ASRK_KV_PAGE == 0) return -1;
    const int page = c.table[slot * c.max_pages + len / ASRK_KV_PAGE];
    return page < c.num_pages ? page : -1;
}

__device__ __forceinline__ int load_agent(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Scratch of the page kernels, in the caller's zero-initialised buffer (every call leaves the first two zero again).
struct Scratch {
    int *writers, *lowest, *list, *tmp, *moves, *count;
    __host__ __device__ Scratch(int32_t* p, int64_t pages, int64_t slots) {
        writers = p;               // [pages] sequences that write into the page
        lowest = writers + pages;  // [pages] (slots - index) of the first of them
        list = lowest + pages;     // [pages] pages to hand out / new number of a page
        tmp = list + pages;        // [slots][2]
        moves = tmp + 2 * slots;   // [max(slots, pages)][2] page copies: source, target
        count = moves + 2 * (slots > pages ? slots : pages);
    }
};

// The holders of four pages from `at` on.
constexpr int LIST_PER = 4;
struct Refs {
    int r[LIST_PER];
    __device__ __forceinline__ void load(const int* refs, int at, int to) {
#pragma unroll
        for (int i = 0; i < LIST_PER; ++i) r[i] = at + i < to ? refs[at + i] : -1;
    }
};

// Lists up to `want` pages, in ascending order from `from` (below `to`), whose holders are none (FREE) or some: put(place, page);
// returns how many there are.  `held`: of this thread's pages from `from` on.
template <bool FREE, class Put>
__device__ __forceinline__ int list_pages(const int* refs, Refs held, int from, int to, int want, int* lds, Put&& put) {
    int found = 0;
    for (int base = from; base < to && found < want; base += MANAGE_T * LIST_PER) {
        const int at = base + threadIdx.x * LIST_PER;
        if (base > from) held.load(refs, at, to);
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < LIST_PER; ++i) mine |= (FREE ? held.r[i] == 0 : held.r[i] > 0) ? 1u << i : 0;
        int total;
        int r = found + block_scan_exclusive(__popc(mine), lds, total);
        for (; mine && r < want; mine &= mine - 1, ++r) put(r, at + __builtin_ctz(mine));
        found += total;
    }
    return found < want ? found : want;
}

// Room for n[s] more tokens of every sequence: the lowest free pages, in the order of the sequences, and a page of its
// own for a sequence that writes into one it shares -- the first of its holders keeps it if they all write.  All or
// nothing: without enough pages (or with a count that does not fit) nothing is added and `status` says so.  One
// workgroup: the work is a few integers per sequence and the order has to be total.  Bound by its chain of dependent accesses
// and by instructions that are fetched for the first time (the cache for them is cold: 1 to 1.5 us per KB of code that runs).
// So a sequence per thread (SMALL) is held in registers and LDS from one step to the next, the first pages' holders are on
// their way from the start, and nothing is unrolled that need not be: 3.7 us for a step of 5 sequences, 4.8 of 160 that share
// their pages (through memory, and with twice the code, 7 and 10), once per step for all layers.
template <bool SMALL>  // at most MANAGE_T sequences
__global__ __launch_bounds__(MANAGE_T) void kv_extend_kernel(asrk_kv_cache c, const int* __restrict__ n_each, int n_all) {
    __shared__ int lds[MANAGE_T / 64];
    __shared__ int shared_page[SMALL ? 2 * MANAGE_T : 1], writers[SMALL ? 2 * MANAGE_T : 1], lowest[SMALL ? 2 * MANAGE_T : 1];  // hashed, -1: none
    __shared__ int fresh[MANAGE_T];  // the pages handed out, if they are few
    __shared__ int flags, n_moves;
    Scratch sc(c.scratch, c.num_pages, (int64_t)c.num_seqs * c.seq_stride);
    const int S = c.num_seqs, M = c.max_pages;
    struct Seq {
        int len, n, page, refs;  // page: the open one, if it is written into
    };
    auto load = [&](int s) -> Seq {
        const int64_t slot = (int64_t)s * c.seq_stride;
        Seq q{c.lens[slot], n_each ? n_each[s] : n_all, -1, 0};
        if (q.n > 0 && q.n <= M * ASRK_KV_PAGE - q.len) q.page = open_page(c, slot, q.len);
        if (q.page >= 0) q.refs = c.refs[q.page];
        return q;
    };
    Refs first;
    first.load(c.refs, threadIdx.x * LIST_PER, c.num_pages);
    if (threadIdx.x == 0) { flags = 0; n_moves = 0; }
    Seq mine{0, 0, -1, 0};
    if (SMALL && (int)threadIdx.x < S) mine = load(threadIdx.x);
    auto seq = [&](int s) -> Seq { return SMALL ? mine : load(s); };
    if (SMALL)
#pragma unroll
        for (int i = 0; i < 2 * MANAGE_T; i += MANAGE_T) {
            shared_page[i + threadIdx.x] = -1;
            writers[i + threadIdx.x] = lowest[i + threadIdx.x] = 0;
        }
    __syncthreads();
    int place = 0;
    if (SMALL && mine.refs > 1) {  // at most half of the places are taken
        place = (uint32_t)mine.page * 0x9e3779b1u >> 21;
        for (;; place = (place + 1) % (2 * MANAGE_T)) {
            const int there = atomicCAS(&shared_page[place], -1, mine.page);
            if (there == -1 || there == mine.page) break;
        }
        atomicAdd(&writers[place], 1);
        atomicMax(&lowest[place], S - (int)threadIdx.x);
    }
    for (int s = threadIdx.x; s < S; s += MANAGE_T) {  // who writes into which open page
        const Seq q = seq(s);
        if (q.n < 0) atomicOr(&flags, ASRK_KV_BAD_COUNT);
        else if (q.n > M * ASRK_KV_PAGE - q.len) atomicOr(&flags, ASRK_KV_TOO_LONG);
        else if (!SMALL && q.page >= 0) {
            atomicAdd(&sc.writers[q.page], 1);
            atomicMax(&sc.lowest[q.page], S - s);
        }
    }
    __syncthreads();  // one workgroup: its atomics are done (at L2) and are read there, past L1
    const bool fits = flags == 0;
    int need_all = 0, my_begin = 0, my_copy = 0;
    for (int base = 0; base < S && fits; base += MANAGE_T) {
        const int s = base + threadIdx.x;
        int need = 0, copy = 0;
        if (s < S) {
            const Seq q = seq(s);
            need = (q.len + q.n + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE - (q.len + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE;
            if (q.page >= 0 && q.refs > 1) {
                const int all = SMALL ? writers[place] : load_agent(&sc.writers[q.page]);
                const int lead = SMALL ? lowest[place] : load_agent(&sc.lowest[q.page]);
                copy = !(all == q.refs && lead == S - s);
            }
            need += copy;
        }
        int total;
        const int begin = need_all + block_scan_exclusive(need, lds, total);
        if (SMALL) {
            my_begin = begin;
            my_copy = copy;
        } else if (s < S) {
            sc.tmp[2 * s] = begin;
            sc.tmp[2 * s + 1] = copy;
        }
        need_all += total;
    }
    int got = 0;
    const bool few = need_all <= MANAGE_T;
    if (fits && need_all > 0) {
        got = need_all <= c.num_pages ? list_pages<true>(c.refs, first, 0, c.num_pages, need_all, lds,
                                                         [&](int r, int page) {
                                                             if (few) fresh[r] = page;
                                                             else sc.list[r] = page;
                                                         })
                                      : 0;
        if (got < need_all && threadIdx.x == 0) flags = ASRK_KV_OUT_OF_PAGES;
        __syncthreads();
    }
    const bool go = fits && got == need_all;
    auto handed = [&](int i) { return few ? fresh[i] : load_agent(&sc.list[i]); };
    for (int s = threadIdx.x; s < S; s += MANAGE_T) {
        const int64_t slot = (int64_t)s * c.seq_stride;
        const Seq q = seq(s);
        const int begin = SMALL ? my_begin : sc.tmp[2 * s], copy = SMALL ? my_copy : sc.tmp[2 * s + 1];
        int* row = c.table + slot * M;
        if (!SMALL && q.page >= 0) {
            sc.writers[q.page] = 0;
            sc.lowest[q.page] = 0;
        }
        if (go) {
            if (copy) {
                const int own = handed(begin);
                row[q.len / ASRK_KV_PAGE] = own;
                c.refs[own] = 1;
                atomicSub(&c.refs[q.page], 1);
                const int m = atomicAdd(&n_moves, 1);
                sc.moves[2 * m] = q.page;
                sc.moves[2 * m + 1] = own;
            }
            int at = begin + copy;
            for (int j = (q.len + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE; j < (q.len + q.n + ASRK_KV_PAGE - 1) / ASRK_KV_PAGE; ++j, ++at) {
                const int own = handed(at);
                row[j] = own;
                c.refs[own] = 1;
            }
            c.lens[slot] = q.len + q.n;
        }
        c.starts[slot] = q.len;  // also if nothing was added: then no row is new
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sc.count[0] = n_moves;
        if (flags) c.status[0] |= flags;
    }
}

// The pages of a list (source, target), every layer: bytes and scales.  HBM-bound: 128 pages of 32 layers (335 MB read and
// written) 55 us = 6.1 TB/s, 289 pages (757 MB) 160 us = 4.7 TB/s; 4 us where the list is empty.
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(asrk_kv_cache c) {
    const Scratch sc(c.scratch, c.num_pages, (int64_t)c.num_seqs * c.seq_stride);
    const int n = sc.count[0];
    const int64_t vecs = (int64_t)c.kv_heads * 2 * ASRK_KV_PAGE * c.head_dim / 16;  // 16-byte pieces of a page of one layer
    const int64_t layer = (int64_t)blockIdx.y * c.num_pages;
    for (int m = blockIdx.x; m < n; m += gridDim.x) {
        const int64_t src = layer + sc.moves[2 * m], dst = layer + sc.moves[2 * m + 1];
        const u32x4* a = (const u32x4*)c.kv + src * vecs;
        u32x4* b = (u32x4*)c.kv + dst * vecs;
        for (int64_t i = threadIdx.x + (int64_t)blockIdx.z * 256; i < vecs; i += 256 * gridDim.z) b[i] = a[i];
        if (blockIdx.z == 0)
            for (int h = threadIdx.x; h < c.kv_heads; h += 256) ((int*)c.exps)[dst * c.kv_heads + h] = ((const int*)c.exps)[src * c.kv_heads + h];
    }
}

// Beam k of group b goes on from beam parents[b][k] of the same group (-1: from nothing, its pages are given back).
// A workgroup owns some columns of the group's table rows, a thread one entry: all is read before anything is written, in place,
// in one launch (1.7 us for 5 sequences, 4.8 for 160; a thread per column with its beams unrolled, 16 times the code, 4.0 and 6.4).
constexpr int REORDER_MAX = 32;
__global__ __launch_bounds__(1024) void kv_reorder_kernel(asrk_kv_cache c, const int64_t* __restrict__ parents, int K, int log_columns) {
    const int b = blockIdx.y, k = threadIdx.x >> log_columns, j = (blockIdx.x << log_columns) + (threadIdx.x & ((1 << log_columns) - 1));
    const int64_t par = parents[(int64_t)b * K + k], first = (int64_t)b * K * c.seq_stride;
    const bool known = par >= 0 && par < K, gone = par == -1;
    const int64_t slot = first + (int64_t)k * c.seq_stride, from = known ? first + par * c.seq_stride : slot;
    int* entry = c.table + slot * c.max_pages + j;
    int now = -1, then = -1, len = 0;
    if (j < c.max_pages) {
        now = *entry;
        then = gone ? -1 : c.table[from * c.max_pages + j];
    }
    if (j == 0 && !gone) len = c.lens[from];
    __syncthreads();
    if (now != then) {
        *entry = then;
        if (then >= 0) atomicAdd(&c.refs[then], 1);
        if (now >= 0) atomicSub(&c.refs[now], 1);
    }
    if (j == 0) {
        if (!known && !gone) atomicOr(&c.status[0], ASRK_KV_BAD_PARENT);
        c.lens[slot] = len;
        c.starts[slot] = len;  // no token is new: a write before the next extend could meet a shared page
    }
}

// Compaction: the r-th page in use at or above the number of pages in use goes to the r-th free one below it, so
// sources and targets are disjoint and all copies run at once.
__global__ __launch_bounds__(MANAGE_T) void kv_compact_plan_kernel(asrk_kv_cache c) {
    __shared__ int lds[MANAGE_T / 64];
    Scratch sc(c.scratch, c.num_pages, (int64_t)c.num_seqs * c.seq_stride);
    const int P = c.num_pages;
    int mine = 0, used;
    for (int p = threadIdx.x; p < P; p += MANAGE_T) {
        mine += c.refs[p] > 0;
        sc.list[p] = p;
    }
    block_scan_exclusive(mine, lds, used);
    int* holes = sc.writers;  // both are zero between calls; they are cleared again below
    int* high = sc.lowest;
    Refs first;
    first.load(c.refs, threadIdx.x * LIST_PER, used);
    const int n = list_pages<true>(c.refs, first, 0, used, used, lds, [&](int r, int page) { holes[r] = page; });
    first.load(c.refs, used + threadIdx.x * LIST_PER, P);
    list_pages<false>(c.refs, first, used, P, n, lds, [&](int r, int page) { high[r] = page; });
    __syncthreads();
    for (int r = threadIdx.x; r < n; r += MANAGE_T) {
        const int src = load_agent(&high[r]), dst = load_agent(&holes[r]);
        sc.moves[2 * r] = src;
        sc.moves[2 * r + 1] = dst;
        sc.list[src] = dst;
        c.refs[dst] = c.refs[src];
        c.refs[src] = 0;
    }
    __syncthreads();
    for (int r = threadIdx.x; r < n; r += MANAGE_T) {
        holes[r] = 0;
        high[r] = 0;
    }
    if (threadIdx.x == 0) {
        sc.count[0] = n;
        c.status[1] = used;
    }
}
__global__ __launch_bounds__(256) void kv_rename_kernel(asrk_kv_cache c) {
    const Scratch sc(c.scratch, c.num_pages, (int64_t)c.num_seqs * c.seq_stride);
    const int64_t n = (int64_t)c.num_seqs * c.seq_stride * c.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int p = c.table[i];
        if (p >= 0) {
            const int q = sc.list[p];
            if (q != p) c.table[i] = q;
        }
    }
}

// ---- tokens in

template <class T>
struct Eight;  // eight values as they are loaded
template <>
struct Eight<float> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const f32x4*>(p)[0]; b = reinterpret_cast<const f32x4*>(p)[1]; }
    __device__ __forceinline__ float operator[](int i) const { return i < 4 ? a[i] : b[i - 4]; }
    __device__ __forceinline__ uint32_t most() const {  // the largest magnitude, as bits: from 0x7f800000 on, something is not finite
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = __float_as_uint((*this)[i]) & 0x7fffffffu;
            m = x > m ? x : m;
        }
        return m;
    }
};
template <>
struct Eight<bf16_t> {
    bf16x8 a;
    __device__ __forceinline__ void load(const bf16_t* p) { a = *reinterpret_cast<const bf16x8*>(p); }
    __device__ __forceinline__ float operator[](int i) const { return (float)a[i]; }
    __device__ __forceinline__ uint32_t most() const {  // two by two, as integers
        typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
        const u32x4 w = __builtin_bit_cast(u32x4, a);
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        return (uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16;
    }
};

__device__ __forceinline__ int exponent_of(float most) {  // smallest e with most <= 448 2^e, clamped
    const uint32_t b = __float_as_uint(most);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b == 0 ? ASRK_KV_EXP_MIN : (e < ASRK_KV_EXP_MIN ? ASRK_KV_EXP_MIN : (e > ASRK_KV_EXP_MAX ? ASRK_KV_EXP_MAX : e));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // normal range only

// four values / scale -> four e4m3 bytes, to the nearest, ties to even; not finite: NaN
__device__ __forceinline__ uint32_t to_e4m3x4(float x0, float x1, float x2, float x3, float inv) {
    const float x[4] = {x0, x1, x2, x3};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -448.f, 448.f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    uint32_t u = (uint32_t)w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(fabsf(x[i]) < __builtin_inff())) u |= 0x7fu << (8 * i);
    return u;
}
// the same where all of them are finite and none is larger than 448 / inv
__device__ __forceinline__ uint32_t plain_e4m3x4(float x0, float x1, float x2, float x3, float inv) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0 * inv, x1 * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2 * inv, x3 * inv, w, true);
}
// the same of two numbers, already divided
__device__ __forceinline__ uint32_t to_e4m3x2(float x0, float x1) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(x0, -448.f, 448.f), __builtin_amdgcn_fmed3f(x1, -448.f, 448.f), 0, false);
    return w | (fabsf(x0) < __builtin_inff() ? 0u : 0x7fu) | (fabsf(x1) < __builtin_inff() ? 0u : 0x7f00u);
}
// four e4m3 bytes times 2^shift (shift <= 0), rounded again
__device__ __forceinline__ uint32_t shift_e4m3x4(uint32_t u, float factor) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    return to_e4m3x4(a[0], a[1], b[0], b[1], factor);
}

// What a page's scales become with new tokens from t0 on, whose largest magnitudes are mk and mv, and the factors of its older ones.
struct Scales {
    int ek, ev, flag;
    float fk = 1.f, fv = 1.f;
    __device__ __forceinline__ Scales(int old, int t0, float mk, float mv, bool odd) : ek(exponent_of(mk)), ev(exponent_of(mv)), flag(odd) {
        if (t0 > 0) {
            const int ok = (int8_t)old, ov = (int8_t)(old >> 8);
            ek = ek > ok ? ek : ok;
            ev = ev > ov ? ev : ov;
            fk = pow2(ok - ek > -60 ? ok - ek : -60);  // 448 2^-60 is zero in e4m3 as well
            fv = pow2(ov - ev > -60 ? ov - ev : -60);
            flag |= (old >> 16) & 1;
        }
    }
    __device__ __forceinline__ int word() const { return (ek & 0xff) | ((ev & 0xff) << 8) | (flag << 16); }
};

// One token: a wave per (head, sequence), a lane per d (D 128: two).  Latency: lengths -> page number -> scales -> stores, and
// little code; the bytes of the values' column are stored one by one, which needs no read.  320 sequences of 5 heads 5.1 us (the
// kernel below with one wave, which turns four tokens at a time and reads the others first, 7.5).
template <class T, int D>
__global__ __launch_bounds__(64) void kv_write_one_kernel(asrk_kv_cache c, const T* __restrict__ k, const T* __restrict__ v, int64_t seq_ld,
                                                          int64_t head_ld, int64_t layer) {
    constexpr int U = D / 64;
    const int h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x;
    const int64_t row = (int64_t)s * seq_ld + (int64_t)h * head_ld + lane, slot = (int64_t)s * c.seq_stride;
    const int start = c.starts[slot], len = c.lens[slot];
    float kx[U], vx[U], mk = 0.f, mv = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        kx[u] = (float)k[row + 64 * u];
        vx[u] = (float)v[row + 64 * u];
    }
    const int pj = start / ASRK_KV_PAGE, t = start % ASRK_KV_PAGE;
    if (len <= start || pj >= c.max_pages) return;
    const int page = c.table[slot * c.max_pages + pj];
    if (page < 0 || page >= c.num_pages) return;
    const int64_t at = (layer * c.num_pages + page) * c.kv_heads + h;
    uint8_t* kp = (uint8_t*)c.kv + at * 2 * ASRK_KV_PAGE * D;
    uint8_t* vp = kp + ASRK_KV_PAGE * D;
    int* ep = (int*)c.exps + at;
    const int old = *ep;
    bool odd = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        mk = fabsf(kx[u]) < __builtin_inff() ? fmaxf(mk, fabsf(kx[u])) : mk;
        mv = fabsf(vx[u]) < __builtin_inff() ? fmaxf(mv, fabsf(vx[u])) : mv;
        odd |= !(fabsf(vx[u]) < __builtin_inff());
    }
    const Scales sc(old, t, __uint_as_float(wave_imax(__float_as_uint(mk))), __uint_as_float(wave_imax(__float_as_uint(mv))), __any(odd));
    if (sc.fk != 1.f)
        for (int u = lane; u < t * D / 4; u += 64) ((uint32_t*)kp)[u] = shift_e4m3x4(((const uint32_t*)kp)[u], sc.fk);
    if (sc.fv != 1.f)
        for (int u = lane; u < D; u += 64)
            for (int g = 0; g < (t + 3) / 4; ++g) {  // by the lane that stores the new byte of this row, in front of it
                uint32_t* p = reinterpret_cast<uint32_t*>(vp + u * ASRK_KV_PAGE) + g;
                *p = shift_e4m3x4(*p, sc.fv);
            }
    const float ik = pow2(-sc.ek), iv = pow2(-sc.ev);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int d = lane + 64 * u;
        const uint32_t two = to_e4m3x2(kx[u] * ik, vx[u] * iv);
        kp[t * D + d] = (uint8_t)two;
        vp[d * ASRK_KV_PAGE + t] = (uint8_t)(two >> 8);
    }
    if (lane == 0) *ep = sc.word();
}

// One workgroup per (head, page that new tokens touch, sequence).  The new rows are read once, into registers: the largest
// magnitude first (as integers, bf16 two by two), then the bytes; what is not finite, or saturates, takes a path of its own.  Value
// bytes are turned through LDS four by four (rows of D + 4 bytes: 16 x 4 lanes read different banks).  Older tokens of the page
// are only touched if the exponent grows.  Heads vary fastest over the grid: neighbours read, and the rows are whole, together.
// 16 prompts of up to 1541 tokens, 5 heads of 64 9.6 us; with every value looked at as fp32 13.6.
template <class T, int D>
__global__ __launch_bounds__(256) void kv_write_kernel(asrk_kv_cache c, const T* __restrict__ k, const T* __restrict__ v, int64_t seq_ld,
                                                           int64_t row_ld, int64_t head_ld, int n, int64_t layer) {
    constexpr int THREADS = 256, PER = D / 8, LINE = D + 4, U = ASRK_KV_PAGE * PER / THREADS;  // U pieces of eight values per thread and tensor
    __shared__ __attribute__((aligned(16))) uint8_t turn[ASRK_KV_PAGE * LINE];
    __shared__ __attribute__((aligned(16))) int most[2][4];
    const int H = c.kv_heads, M = c.max_pages;
    const int s = blockIdx.z, h = blockIdx.x;
    const int64_t slot = (int64_t)s * c.seq_stride;
    const int start = c.starts[slot];
    int rows = c.lens[slot] - start;
    rows = rows < n ? rows : n;
    const int pj = start / ASRK_KV_PAGE + blockIdx.y;
    const int lo = start > pj * ASRK_KV_PAGE ? start : pj * ASRK_KV_PAGE;
    const int hi = start + rows < (pj + 1) * ASRK_KV_PAGE ? start + rows : (pj + 1) * ASRK_KV_PAGE;
    if (lo >= hi || pj >= M) return;
    const int page = c.table[slot * M + pj];
    const int t0 = lo - pj * ASRK_KV_PAGE, t1 = hi - pj * ASRK_KV_PAGE;  // new tokens of this page: [t0, t1)
    const int64_t base = (int64_t)s * seq_ld + (int64_t)h * head_ld - (int64_t)(start - pj * ASRK_KV_PAGE) * row_ld;  // row of token t: base + t * row_ld
    const int units = (t1 - t0) * PER;
    Eight<T> kx[U], vx[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int u = j * THREADS + threadIdx.x;
        if (u < units) {
            const int64_t o = base + (int64_t)(t0 + u / PER) * row_ld + u % PER * 8;
            kx[j].load(k + o);
            vx[j].load(v + o);
        }
    }
    if (page < 0 || page >= c.num_pages) return;
    const int64_t at = ((layer * c.num_pages + page) * H + h);
    uint8_t* kp = (uint8_t*)c.kv + at * 2 * ASRK_KV_PAGE * D;
    uint8_t* vp = kp + ASRK_KV_PAGE * D;
    int8_t* ep = c.exps + at * 4;
    const int old = *reinterpret_cast<const int*>(ep);
    constexpr int INF = 0x7f800000;
    int mk = 0, mv = 0;  // magnitudes as bits
    auto over_workgroup = [&]() __attribute__((always_inline)) {
        mk = wave_imax(mk);
        mv = wave_imax(mv);
        most[0][threadIdx.x >> 6] = mk;
        most[1][threadIdx.x >> 6] = mv;
        __syncthreads();
        const int4 a = *reinterpret_cast<const int4*>(most[0]), b = *reinterpret_cast<const int4*>(most[1]);
        mk = larger(larger(a.x, a.y), larger(a.z, a.w));
        mv = larger(larger(b.x, b.y), larger(b.z, b.w));
    };
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (j * THREADS + (int)threadIdx.x < units) {
            mk = larger(mk, kx[j].most());
            mv = larger(mv, vx[j].most());
        }
    over_workgroup();
    const bool odd = mv >= INF, special = odd || mk >= INF;
    if (special) {  // rare: once more, of the finite ones
        mk = mv = 0;
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (j * THREADS + (int)threadIdx.x < units) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int x = __float_as_uint(kx[j][i]) & 0x7fffffff, y = __float_as_uint(vx[j][i]) & 0x7fffffff;
                    mk = x < INF ? larger(mk, x) : mk;
                    mv = y < INF ? larger(mv, y) : mv;
                }
            }
        __syncthreads();  // `most` has been read
        over_workgroup();
    }
    const Scales sc(old, t0, __uint_as_float(mk), __uint_as_float(mv), odd);
    const float ik = pow2(-sc.ek), iv = pow2(-sc.ev);
    if (sc.fk != 1.f)
        for (int u = threadIdx.x; u < t0 * D / 4; u += THREADS) ((uint32_t*)kp)[u] = shift_e4m3x4(((const uint32_t*)kp)[u], sc.fk);
    auto convert = [&](auto&& four) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int u = j * THREADS + threadIdx.x;
            if (u < units) {
                const int t = t0 + u / PER, d = u % PER * 8;
                u32x2 w;
                w[0] = four(kx[j][0], kx[j][1], kx[j][2], kx[j][3], ik);
                w[1] = four(kx[j][4], kx[j][5], kx[j][6], kx[j][7], ik);
                *reinterpret_cast<u32x2*>(kp + t * D + d) = w;
                uint32_t* line = reinterpret_cast<uint32_t*>(turn + t * LINE + d);
                line[0] = four(vx[j][0], vx[j][1], vx[j][2], vx[j][3], iv);
                line[1] = four(vx[j][4], vx[j][5], vx[j][6], vx[j][7], iv);
            }
        }
    };
    if (special || sc.ek == ASRK_KV_EXP_MAX || sc.ev == ASRK_KV_EXP_MAX) convert(to_e4m3x4);
    else convert(plain_e4m3x4);
    __syncthreads();
    // four tokens by four d's per step; lanes run over the tokens first, so that stores are whole lines
    const bool shift = sc.fv != 1.f;
    for (int u = threadIdx.x; u < 16 * (D / 4); u += THREADS) {
        const int g = u % 16, d = u / 16 * 4;
        if (g * 4 >= t1 || (!shift && g * 4 + 4 <= t0)) continue;
        uint32_t w[4], x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(turn + (g * 4 + i) * LINE + d);  // token 4 g + i: d .. d + 3
        const uint32_t a0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), a1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
        const uint32_t b0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), b1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
        x[0] = __builtin_amdgcn_perm(b0, a0, 0x05040100);  // d: tokens 4 g .. 4 g + 3
        x[1] = __builtin_amdgcn_perm(b0, a0, 0x07060302);
        x[2] = __builtin_amdgcn_perm(b1, a1, 0x05040100);
        x[3] = __builtin_amdgcn_perm(b1, a1, 0x07060302);
        uint32_t mask = 0;  // of the new tokens among the four
#pragma unroll
        for (int i = 0; i < 4; ++i) mask |= g * 4 + i >= t0 && g * 4 + i < t1 ? 0xffu << (8 * i) : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = 0;
        if (mask != 0xffffffffu)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(vp + (d + i) * ASRK_KV_PAGE + g * 4) & ~mask;
        if (shift)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = shift_e4m3x4(w[i], sc.fv);
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(vp + (d + i) * ASRK_KV_PAGE + g * 4) = (x[i] & mask) | w[i];
    }
    if (threadIdx.x == 0) *reinterpret_cast<int*>(ep) = sc.word();
}
template <class T, int D>
void launch_write(const asrk_kv_cache* c, const void* k, const void* v, int64_t seq_ld, int64_t row_ld, int64_t head_ld, int n, int layer,
                  hipStream_t st) {
    if (n == 1) {
        hipLaunchKernelGGL((kv_write_one_kernel<T, D>), dim3(c->kv_heads, c->num_seqs), dim3(64), 0, st, *c, (const T*)k, (const T*)v, seq_ld,
                           head_ld, (int64_t)layer);
        return;
    }
    const dim3 grid(c->kv_heads, (unsigned)(((int64_t)n + ASRK_KV_PAGE - 2) / ASRK_KV_PAGE + 1), c->num_seqs);
    hipLaunchKernelGGL((kv_write_kernel<T, D>), grid, dim3(256), 0, st, *c, (const T*)k, (const T*)v, seq_ld, row_ld, head_ld, n, (int64_t)layer);
}

// ---- tokens out

// One workgroup per (page, head, layer and sequence) of the tokens [first, first + count) of every sequence.  Both pages are
// loaded at once; the value page is turned through LDS (rows of 68 bytes: 8 x 8 lanes read different banks), two tokens of eight d's
// per step.  HBM-bound: 25600 pages (629 MB) 120 us = 5.2 TB/s; with the heads slowest over the grid, whose lines of a row are then
// written far apart in time, a third more.
template <int D>
__global__ __launch_bounds__(256) void kv_read_kernel(asrk_kv_cache c, const int* __restrict__ first_each, int first_all, int count,
                                                      int layer0, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out) {
    constexpr int PER = D / 8, UK = ASRK_KV_PAGE * PER / 256, UV = D * ASRK_KV_PAGE / 16 / 256;
    __shared__ uint32_t turn[D * 17];
    const int H = c.kv_heads, M = c.max_pages;
    const int h = blockIdx.x;
    int s = blockIdx.z, l = 0;
    if ((int)gridDim.z != c.num_seqs) {
        l = (unsigned)s / (unsigned)c.num_seqs;
        s -= l * c.num_seqs;
    }
    const int64_t slot = (int64_t)s * c.seq_stride;
    const int64_t first = first_each ? first_each[s] : first_all;
    const int64_t pj = (first >> 6) + blockIdx.y;  // pages of 64, also of what lies in front of the sequence
    const int64_t t_lo = first - pj * ASRK_KV_PAGE, t_hi = first + count - pj * ASRK_KV_PAGE;  // asked tokens within the page
    if (t_hi <= 0) return;
    const int lo = t_lo > 0 ? (int)t_lo : 0, hi = t_hi < ASRK_KV_PAGE ? (int)t_hi : ASRK_KV_PAGE;
    if (lo >= hi) return;
    int have = 0, page = -1;  // tokens that the page has
    if (pj >= 0 && pj < M) {
        const int64_t left = c.lens[slot] - pj * ASRK_KV_PAGE;
        page = c.table[slot * M + pj];
        have = page >= 0 && page < c.num_pages && left > 0 ? (left < ASRK_KV_PAGE ? (int)left : ASRK_KV_PAGE) : 0;
    }
    const int64_t at = (((int64_t)(layer0 + l) * c.num_pages + (have ? page : 0)) * H + h);
    const uint8_t* kp = (const uint8_t*)c.kv + at * 2 * ASRK_KV_PAGE * D;
    const uint8_t* vp = kp + ASRK_KV_PAGE * D;
    const int e = *reinterpret_cast<const int*>(c.exps + at * 4);
    u32x2 kx[UK];
    u32x4 vx[UV];
    if (have) {
#pragma unroll
        for (int j = 0; j < UV; ++j) vx[j] = reinterpret_cast<const u32x4*>(vp)[j * 256 + threadIdx.x];
#pragma unroll
        for (int j = 0; j < UK; ++j) kx[j] = reinterpret_cast<const u32x2*>(kp)[j * 256 + threadIdx.x];
#pragma unroll
        for (int j = 0; j < UV; ++j) {
            const int u = j * 256 + threadIdx.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) turn[(u >> 2) * 17 + (u & 3) * 4 + i] = vx[j][i];
        }
    }
    __syncthreads();
    const float sk = pow2((int8_t)e), sv = pow2((int8_t)(e >> 8));
    const int64_t out0 = (((int64_t)l * c.num_seqs + s) * count - t_lo) * H * D + (int64_t)h * D;  // of token 0 of the page
#pragma unroll
    for (int j = 0; j < UK; ++j) {
        const int u = j * 256 + threadIdx.x, t = u / PER, d = u % PER * 8;
        if (t < lo || t >= hi) continue;
        u32x4 y = {0, 0, 0, 0};
        if (t < have) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kx[j][i], sk, false));
                y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kx[j][i], sk, true));
            }
        }
        *reinterpret_cast<u32x4*>(k_out + out0 + (int64_t)t * H * D + d) = y;
    }
#pragma unroll
    for (int j = 0; j < UK / 2; ++j) {
        const int u = j * 256 + threadIdx.x, t = u / PER * 2, d = u % PER * 8;
        uint32_t two[8];  // tokens t and t + 1 of d + i
#pragma unroll
        for (int i = 0; i < 8; ++i)
            two[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(turn[(d + i) * 17 + t / 4] >> (8 * (t & 2)), sv, false));
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            if (t + o < lo || t + o >= hi) continue;
            u32x4 y = {0, 0, 0, 0};
            if (t + o < have)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_perm(two[2 * i + 1], two[2 * i], o ? 0x07060302 : 0x05040100);
            *reinterpret_cast<u32x4*>(v_out + out0 + (int64_t)(t + o) * H * D + d) = y;
        }
    }
}

}  // namespace

int asrk_kv_check(const asrk_kv_cache* c) {
    if (!c || !c->kv || !c->exps || !c->table || !c->lens || !c->starts || !c->refs || !c->status || !c->scratch) return ASRK_ERR_NULL;
    if (c->num_layers <= 0 || c->num_pages <= 0 || c->kv_heads <= 0 || c->num_seqs <= 0 || c->max_pages <= 0 || c->seq_stride <= 0)
        return ASRK_ERR_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128) return ASRK_ERR_SHAPE;
    if (c->num_layers > 65535 || c->kv_heads > 65535 || c->num_seqs > 65535 || (int64_t)c->num_seqs * c->seq_stride > 0x7fffffff ||
        (int64_t)c->num_seqs * c->seq_stride * c->max_pages > 0x7fffffff || c->max_pages > 0x7fffffff / ASRK_KV_PAGE ||
        c->num_pages > 0x3fffffff)
        return ASRK_ERR_SHAPE;
    if (((uintptr_t)c->kv & 15) || ((uintptr_t)c->exps & 15) || ((uintptr_t)c->table & 3) || ((uintptr_t)c->lens & 3) ||
        ((uintptr_t)c->starts & 3) || ((uintptr_t)c->refs & 15) || ((uintptr_t)c->status & 3) || ((uintptr_t)c->scratch & 15))
        return ASRK_ERR_ALIGN;
    return ASRK_OK;
}

extern "C" size_t asrk_kv_scratch_bytes(int num_pages, int num_slots) {
    if (num_pages <= 0 || num_slots <= 0) return 0;
    Scratch sc((int32_t*)nullptr, num_pages, num_slots);
    return (size_t)(sc.count + 4 - (int*)nullptr) * sizeof(int32_t);
}

static void launch_copies(const asrk_kv_cache* c, int most, hipStream_t st) {
    const int64_t bytes = (int64_t)c->kv_heads * 2 * ASRK_KV_PAGE * c->head_dim;
    const int parts = (int)((bytes + 16383) / 16384);  // 16 KiB per workgroup and page
    hipLaunchKernelGGL(kv_copy_pages_kernel, dim3(most < 512 ? most : 512, c->num_layers, parts < 64 ? parts : 64), dim3(256), 0, st, *c);
}

extern "C" int asrk_kv_extend(const asrk_kv_cache* c, const int32_t* n_each, int n_all, void* stream) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (!n_each && n_all < 0) return ASRK_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    if (c->num_seqs <= MANAGE_T) hipLaunchKernelGGL(kv_extend_kernel<true>, dim3(1), dim3(MANAGE_T), 0, st, *c, n_each, n_all);
    else hipLaunchKernelGGL(kv_extend_kernel<false>, dim3(1), dim3(MANAGE_T), 0, st, *c, n_each, n_all);
    launch_copies(c, c->num_seqs, st);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}

extern "C" int asrk_kv_reorder(const asrk_kv_cache* c, const int64_t* parents, int K, void* stream) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (!parents) return ASRK_ERR_NULL;
    if (K <= 0 || K > REORDER_MAX || c->num_seqs % K) return ASRK_ERR_SHAPE;
    const int log_columns = K <= 16 ? 6 : 5, columns = 1 << log_columns;
    hipLaunchKernelGGL(kv_reorder_kernel, dim3((c->max_pages + columns - 1) / columns, c->num_seqs / K), dim3(columns * K), 0, (hipStream_t)stream, *c,
                       parents, K, log_columns);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}

extern "C" int asrk_kv_compact(const asrk_kv_cache* c, void* stream) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (c->seq_stride != 1) return ASRK_ERR_SHAPE;  // every table row has to be renamed
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(kv_compact_plan_kernel, dim3(1), dim3(MANAGE_T), 0, st, *c);
    launch_copies(c, c->num_pages, st);
    const int64_t blocks = ((int64_t)c->num_seqs * c->max_pages + 255) / 256;
    hipLaunchKernelGGL(kv_rename_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, *c);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}

extern "C" int asrk_kv_write(const asrk_kv_cache* c, int layer, const void* k, const void* v, int dtype, int64_t seq_ld, int64_t row_ld,
                             int64_t head_ld, int n, void* stream) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (!k || !v) return ASRK_ERR_NULL;
    if (dtype != ASRK_F32 && dtype != ASRK_BF16) return ASRK_ERR_UNSUPPORTED;
    if (layer < 0 || layer >= c->num_layers || n <= 0 || seq_ld < 0 || row_ld < 0 || head_ld < 0) return ASRK_ERR_SHAPE;
    const int per = dtype == ASRK_F32 ? 4 : 8;  // values in 16 bytes
    if (((uintptr_t)k & 15) || ((uintptr_t)v & 15) || seq_ld % per || row_ld % per || head_ld % per) return ASRK_ERR_ALIGN;
    if (((int64_t)n + ASRK_KV_PAGE - 2) / ASRK_KV_PAGE + 1 > 65535) return ASRK_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ASRK_F32 && c->head_dim == 64) launch_write<float, 64>(c, k, v, seq_ld, row_ld, head_ld, n, layer, st);
    else if (dtype == ASRK_F32) launch_write<float, 128>(c, k, v, seq_ld, row_ld, head_ld, n, layer, st);
    else if (c->head_dim == 64) launch_write<bf16_t, 64>(c, k, v, seq_ld, row_ld, head_ld, n, layer, st);
    else launch_write<bf16_t, 128>(c, k, v, seq_ld, row_ld, head_ld, n, layer, st);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}

extern "C" int asrk_kv_read(const asrk_kv_cache* c, int layer, int layers, const int32_t* first_each, int first_all, int count, void* k_out,
                            void* v_out, void* stream) {
    if (int rc = asrk_kv_check(c)) return rc;
    if (!k_out || !v_out) return ASRK_ERR_NULL;
    if (layer < 0 || layers <= 0 || layer + (int64_t)layers > c->num_layers || count <= 0) return ASRK_ERR_SHAPE;
    if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15)) return ASRK_ERR_ALIGN;
    if ((int64_t)layers * c->num_seqs > 65535) return ASRK_ERR_SHAPE;
    const int64_t parts = ((int64_t)count + ASRK_KV_PAGE - 2) / ASRK_KV_PAGE + 1;  // pages that `count` tokens can touch
    if (parts > 65535) return ASRK_ERR_SHAPE;
    const dim3 grid(c->kv_heads, (unsigned)parts, c->num_seqs * layers);
    auto* const kernel = c->head_dim == 64 ? kv_read_kernel<64> : kv_read_kernel<128>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, *c, first_each, first_all, count, layer, (bf16_t*)k_out, (bf16_t*)v_out);
    return hipGetLastError() == hipSuccess ? ASRK_OK : ASRK_ERR_HIP;
}
