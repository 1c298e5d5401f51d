// gfx950 kernels that build a serving step's tables and write its tokens into
// the cache (include/pmkl_cache.h).
#pragma once

#include "cache_common.hpp"

namespace pmkl_amd {

constexpr int kCacheThreads = 256;

// ---------------------------------------------------------------- tables

struct SlotsParams {
    const int32_t *cached_lens;
    const int32_t *new_lens;
    int32_t *table;
    const int32_t *free_pages;
    const int32_t *free_head;
    int32_t *seq_lens;
    int32_t *query_start;
    int64_t *slots;
    int32_t *free_head_out;
    int64_t table_stride;
    int64_t free_count;
    int64_t tokens;
    int32_t batch;
    int32_t width;
    int32_t log2_page;
};

__device__ __forceinline__ int32_t clamp_i32(int64_t x) { return (int32_t)min(x, (int64_t)INT32_MAX); }

// Request b's first token and first new page are sums over the requests before
// it.  Every workgroup forms all of them, 256 requests at a time (a scan in
// each wave, joined through the LDS), and writes its share: of the requests'
// lengths, of the new table entries and of the slots the blocks of 256 whose
// number is its own modulo the grid.  One launch without a word between the
// workgroups, against a scan and a fill of a launch each; the lengths of 1,024
// requests are 8 KB from the L2.  A block finds its requests by bisection of
// the sums in the LDS.
__global__ __launch_bounds__(kCacheThreads) void cache_slots_kernel(SlotsParams p) {
    constexpr int NT = kCacheThreads;
    __shared__ int64_t token0[NT + 1], page0[NT + 1];   // sums before each request of the 256
    __shared__ int64_t part[2][NT / 64];
    __shared__ int32_t held[NT], first[NT];               // its cached tokens, its first new page
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t me = blockIdx.x, grid = gridDim.x;
    const int ps = 1 << p.log2_page;
    const int64_t head = *p.free_head;
    int64_t tokens = 0, pages = 0;                        // of the requests before these

    const auto page_of_list = [&](int64_t i) -> int32_t {
        i += head;
        return i >= 0 && i < p.free_count ? p.free_pages[i] : -1;
    };
    // the last request of the 256 whose sum is at most i
    const auto find = [](const int64_t *sums, int64_t i) {
        int r = 0;
#pragma unroll
        for (int step = NT / 2; step; step >>= 1)
            if (sums[r + step] <= i) r += step;
        return r;
    };

    for (int base = 0; base < p.batch; base += NT) {
        const int b = base + tid;
        int64_t c = 0, n = 0;
        if (b < p.batch) {
            c = max(p.cached_lens[b], 0);
            n = max(p.new_lens[b], 0);
        }
        const int64_t f = min((c + ps - 1) >> p.log2_page, (int64_t)p.width);
        const int64_t e = min((c + n + ps - 1) >> p.log2_page, (int64_t)p.width);
        const int64_t ti = wave_scan(n, lane), pi = wave_scan(e - f, lane);
        if (base) __syncthreads();                        // the blocks below still read the LDS
        if (lane == 63) {
            part[0][wave] = ti;
            part[1][wave] = pi;
        }
        __syncthreads();
        int64_t tb = tokens, pb = pages;
        for (int w = 0; w < wave; ++w) {
            tb += part[0][w];
            pb += part[1][w];
        }
        token0[tid] = tb + ti - n;
        page0[tid] = pb + pi - (e - f);
        if (tid == NT - 1) {
            token0[NT] = tb + ti;
            page0[NT] = pb + pi;
        }
        held[tid] = (int32_t)c;
        first[tid] = (int32_t)f;
        if (b < p.batch && (base / NT) % grid == me) {
            p.query_start[b] = clamp_i32(tb + ti - n);
            p.seq_lens[b] = clamp_i32(c + n);
        }
        __syncthreads();
        const int64_t t1 = min(token0[NT], p.tokens), p1 = page0[NT];

        // blocks of 256 numbered from the call's first page and token on
        const auto first_block = [&](int64_t i) {
            const int64_t blk = i / NT;
            return blk + (me - blk % grid + grid) % grid;
        };
        for (int64_t blk = first_block(pages); blk * NT < p1; blk += grid) {
            const int64_t i = blk * NT + tid;
            if (i >= pages && i < p1) {
                const int r = find(page0, i);
                p.table[(base + r) * p.table_stride + first[r] + (i - page0[r])] = page_of_list(i);
            }
        }
        for (int64_t blk = first_block(tokens); blk * NT < t1; blk += grid) {
            const int64_t i = blk * NT + tid;
            if (i >= tokens && i < t1) {
                const int r = find(token0, i);
                const int64_t at = held[r] + (i - token0[r]);
                const int64_t w = at >> p.log2_page;
                int32_t page = -1;
                if (w < p.width)
                    page = w >= first[r] ? page_of_list(page0[r] + w - first[r])
                                         : p.table[(base + r) * p.table_stride + w];
                p.slots[i] = page < 0 ? -1 : ((int64_t)page << p.log2_page) + (at & (ps - 1));
            }
        }
        tokens = token0[NT];
        pages = p1;
    }
    for (int64_t i = me * NT + tid; i < p.tokens; i += grid * NT)
        if (i >= tokens) p.slots[i] = -1;
    if (me == 0 && tid == 0) {
        p.query_start[p.batch] = clamp_i32(tokens);
        *p.free_head_out = clamp_i32(head + pages);
    }
}

// ---------------------------------------------------------------- appends

struct AppendParams {
    const void *k;
    const void *v;
    const int64_t *slots;
    CacheParams cache;
    int64_t k_st, k_sh, v_st, v_sh;   // elements
    int64_t tokens;
    int32_t kv_heads;
};

// 2^e, the least e >= -126 with a <= 448 * 2^e (448 = 1.75 * 2^8), for finite a >= 0.
__device__ __forceinline__ float cache_scale_for(float a) {
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);   // biased
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// x / s as an e4m3 operand: s is a power of two unless the caller made it.  What
// is not finite becomes NaN (e4m3 has no infinity, and 448 in its place would
// hide it).
struct CacheQuotient {
    float s, inverse;
    bool exact;
    __device__ explicit CacheQuotient(float scale) : s(scale) {
        exact = (__float_as_uint(s) & 0x7fffff) == 0 && s >= 0x1p-126f;
        inverse = 1.f / s;   // of a power of two in 2^-126 .. 2^127: exact
    }
    __device__ float operator()(float x) const {
        const float y = exact ? x * inverse : x / s;
        return fabsf(x) < INFINITY ? y : __builtin_nanf("");
    }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) CacheVec {
    T v[N];
};

// largest finite magnitude of N values
template <typename T, int N>
__device__ __forceinline__ float finite_max(const CacheVec<T, N> &x, float a) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = fabsf((float)x.v[i]);
        a = fmaxf(a, y < INFINITY ? y : 0.f);
    }
    return a;
}

// codes of a dword times f
__device__ __forceinline__ uint32_t cache_rescale(uint32_t codes, float f) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, r, true);
}

// bytes `from` .. `to` - 1 of a dword whose first byte is number `at`
__device__ __forceinline__ uint32_t byte_mask(int at, int from, int to) {
    const int lo = min(max(from - at, 0), 4), hi = min(max(to - at, 0), 4);
    if (lo >= hi) return 0;
    return (0xffffffffu >> (32 - 8 * (hi - lo))) << (8 * lo);
}

// A wave owns (run, head, keys or values): it reads the run's rows for their
// largest value, then again, out of the caches, for the codes.  A workgroup's
// waves, and blockIdx.y's of the same 64 tokens, share what runs begin among
// these tokens: runs are found on the spot, so the call needs neither the
// requests nor their lengths.  Values are transposed on the way: a lane has two
// columns and 16 tokens of a page, and stores each column's 16 codes as one
// vector, with the codes around the run read first.
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void cache_append_kernel(AppendParams p) {
    constexpr int E = 16 / (int)sizeof(T);      // elements of a vector
    constexpr int LPR = D / E;                    // lanes of a row
    const int lane = threadIdx.x & 63;
    const int log2_page = p.cache.log2_page, ps = 1 << log2_page;
    const int64_t limit = (int64_t)p.cache.pages << log2_page;
    const int64_t w0 = (int64_t)blockIdx.x * 64;

    // the runs that begin here
    const int64_t t = w0 + lane;
    const int64_t slot = t < p.tokens ? p.slots[t] : -1;
    const int64_t before = t > 0 && t < p.tokens ? p.slots[t - 1] : -1;
    const bool leads = slot >= 0 && slot < limit && ((slot & (ps - 1)) == 0 || before != slot - 1);
    const uint64_t leaders = __builtin_amdgcn_ballot_w64(leads);
    const int rank = __builtin_popcountll(leaders & ((1ull << lane) - 1));
    const int items = __builtin_popcountll(leaders) * p.kv_heads * 2;

    const int stride = gridDim.y * (kCacheThreads / 64);
    for (int item = blockIdx.y * (kCacheThreads / 64) + (threadIdx.x >> 6); item < items; item += stride) {
        const int which = item & 1, head = (item >> 1) % p.kv_heads, run = (item >> 1) / p.kv_heads;
        const int leader = __builtin_ctzll(__builtin_amdgcn_ballot_w64(leads && rank == run));
        const int64_t t0 = w0 + leader;
        const int64_t s0 = __shfl(slot, leader);
        const int o = (int)(s0 & (ps - 1));
        const int64_t page = s0 >> log2_page;
        int n = 0;                                // tokens of the run
        while (true) {
            const int i = n + lane;
            const bool in = i < ps - o && t0 + i < p.tokens && p.slots[t0 + i] == s0 + i;
            const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
            if (mask != ~0ull) {
                n += __builtin_ctzll(~mask);
                break;
            }
            n += 64;
        }

        const int64_t st = which ? p.v_st : p.k_st;
        const T *x = which ? (const T *)p.v + t0 * p.v_st + head * p.v_sh : (const T *)p.k + t0 * p.k_st + head * p.k_sh;
        float a = 0.f;
        for (int i = lane / LPR; i < n; i += 64 / LPR)
            a = finite_max(*(const CacheVec<T, E> *)(x + i * st + lane % LPR * E), a);
        a = wave_max(a);

        float *scale = which ? p.cache.v_scale + page * (p.cache.vs_sp / 4) + head * p.cache.vs_sh
                             : p.cache.k_scale + page * (p.cache.ks_sp / 4) + head * p.cache.ks_sh;
        const float was = *scale, need = cache_scale_for(a);
        const bool kept = o > 0 && was > 0.f && was < INFINITY;
        const float now = kept ? fmaxf(was, need) : need;
        const bool grown = kept && now != was;
        const float shrink = was / now;
        const CacheQuotient quotient(now);
        if (lane == 0 && !(kept && now == was)) *scale = now;

        if (which == 0) {
            uint8_t *k = p.cache.k + page * p.cache.k_sp + head * p.cache.k_sh;
            for (int i = lane / LPR; i < n; i += 64 / LPR) {
                const auto r = *(const CacheVec<T, E> *)(x + i * st + lane % LPR * E);
                CacheVec<uint32_t, E / 4> c;
#pragma unroll
                for (int j = 0; j < E / 4; ++j) {
                    int q = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r.v[4 * j]), quotient((float)r.v[4 * j + 1]), 0, false);
                    c.v[j] = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r.v[4 * j + 2]), quotient((float)r.v[4 * j + 3]), q, true);
                }
                *(CacheVec<uint32_t, E / 4> *)(k + (int64_t)(o + i) * p.cache.k_st + lane % LPR * E) = c;
            }
            if (grown)
                for (int i = lane / (D / 4); i < o; i += 64 / (D / 4)) {
                    uint32_t *c = (uint32_t *)(k + (int64_t)i * p.cache.k_st + lane % (D / 4) * 4);
                    *c = cache_rescale(*c, shrink);
                }
        } else {
            uint8_t *v = p.cache.v + page * p.cache.v_sp + head * p.cache.v_sh;
            constexpr int LPC = D / 2;            // lanes that cover the columns, two each
            const int d = lane % LPC * 2;
            for (int g = (grown ? 0 : o / 16) + lane / LPC; g < (o + n + 15) / 16; g += 64 / LPC) {
                uint8_t *c0 = v + (int64_t)d * p.cache.v_sd + g * 16, *c1 = c0 + p.cache.v_sd;
                CacheVec<uint32_t, 4> a0 = *(CacheVec<uint32_t, 4> *)c0, a1 = *(CacheVec<uint32_t, 4> *)c1;
                CacheVec<T, 2> r[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)      // tokens outside the run: one of its own, not used
                    r[i] = *(const CacheVec<T, 2> *)(x + min(max(g * 16 + i - o, 0), n - 1) * st + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = g * 16 + 4 * j;
                    const uint32_t fresh = byte_mask(at, o, o + n), old = byte_mask(at, 0, o);
                    const auto pack = [&](int c) -> uint32_t {
                        int q = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r[4 * j].v[c]), quotient((float)r[4 * j + 1].v[c]), 0, false);
                        return __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r[4 * j + 2].v[c]), quotient((float)r[4 * j + 3].v[c]), q, true);
                    };
                    if (grown) {
                        a0.v[j] = (cache_rescale(a0.v[j], shrink) & old) | (a0.v[j] & ~old);
                        a1.v[j] = (cache_rescale(a1.v[j], shrink) & old) | (a1.v[j] & ~old);
                    }
                    a0.v[j] = (pack(0) & fresh) | (a0.v[j] & ~fresh);
                    a1.v[j] = (pack(1) & fresh) | (a1.v[j] & ~fresh);
                }
                *(CacheVec<uint32_t, 4> *)c0 = a0;
                *(CacheVec<uint32_t, 4> *)c1 = a1;
            }
        }
    }
}

}  // namespace pmkl_amd
