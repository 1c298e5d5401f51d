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
// the sums in the LDS.  Bound by latency: 64 requests of a token each 3.8 us, 512 of
// up to 256 tokens 6.2.
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

// x / s as an e4m3 operand.  s is a power of two unless the caller made it: then
// x (1 / s) is the same.  What is not finite becomes NaN (e4m3 has no infinity,
// and 448 in its place would hide it).
template <bool POWER>
struct CacheQuotient {
    float s;      // POWER: its inverse, exact for 2^-126 .. 2^127
    __device__ explicit CacheQuotient(float scale) : s(POWER ? 1.f / scale : scale) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float y = POWER ? x * s : x / s;
        return fabsf(x) < INFINITY ? y : __builtin_nanf("");
    }
};
__device__ __forceinline__ bool is_power(float s) { return (__float_as_uint(s) & 0x7fffff) == 0 && s >= 0x1p-126f; }

// f(CacheQuotient) for a scale that is the same in the wave
template <typename F>
__device__ __forceinline__ void with_quotient(float scale, F f) {
    if (is_power(scale))
        f(CacheQuotient<true>(scale));
    else
        f(CacheQuotient<false>(scale));
}

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

// N elements as they were loaded: whole words, where the elements by themselves
// would take a register each.  settle() keeps what was made of them (their fp32
// values) from being held beside them.
template <typename T, int N>
struct CacheRaw {
    static constexpr int W = sizeof(T) * N / 4;
    typedef uint32_t words __attribute__((ext_vector_type(W)));
    words w;
    __device__ __forceinline__ void load(const T *p) { w = *(const words *)p; }
    __device__ __forceinline__ CacheVec<T, N> get() const { return __builtin_bit_cast(CacheVec<T, N>, w); }
    __device__ __forceinline__ void settle() { asm volatile("" : "+v"(w)); }
};
template <typename T>
struct CacheRaw<T, 2> {
    static constexpr int W = sizeof(T) * 2 / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p) {
        const CacheVec<uint32_t, W> x = *(const CacheVec<uint32_t, W> *)p;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = x.v[i];
    }
    __device__ __forceinline__ CacheVec<T, 2> get() const { return __builtin_bit_cast(CacheVec<T, 2>, w); }
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
    }
};

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
// largest value and makes the codes of them, from the registers where they fit (a
// run inside one page of 16 or 32), else read again, out of the caches.  A
// workgroup's waves, and blockIdx.y's of the same 64 tokens, share what runs begin
// among these tokens: runs are found on the spot, so the call needs neither the
// requests nor their lengths.  Values are transposed on the way: a lane has two
// columns and 16 tokens of a page, and stores each column's 16 codes as one
// vector, with the codes around the run read first.  Bound by latency: a decoding
// step of 256 requests, bf16, 8 heads of 128, 7.0 us (slots, then rows, scales and codes,
// then stores); 4 prompts of 2,048 tokens, 51 MB, 15.4 us, 3.3 TB/s.
// In pages of 64 tokens and more a wave would read and write for long: where no more
// than three runs begin among the 64 tokens, a workgroup's waves take a (run, head,
// keys or values) together, a share of its rows each, in pages of 64 only while the
// call has few items (together and by a wave each, us: 8 prompts of 1,000 tokens, 8 heads
// of 128, pages of 256 25.2, 40.7; 2 of 500 in pages of 128 7.4, 15.8; 24 requests of 1 to 128
// tokens, pages of 64 6.4, 6.9; but 16 of 64 tokens, 16 heads, pages of 64 7.5, 6.2; 64 of 20
// 9.7, 6.9).
constexpr int kAppendRows = 8;   // vectors of a lane that are kept

template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads, 4) void cache_append_kernel(AppendParams p) {
    constexpr int E = 16 / (int)sizeof(T);      // elements of a vector
    constexpr int LPR = D / E;                    // lanes of a row
    constexpr int NW = kCacheThreads / 64;
    __shared__ float largest[2][NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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

    const bool together = ps >= 64 && __builtin_popcountll(leaders) <= 3 && (ps > 64 || (int64_t)items * gridDim.x <= 640);
    const int sub = together ? wave : 0, of = together ? NW : 1;   // the wave's share
    int turn = 0;
    for (int item = together ? blockIdx.y : blockIdx.y * NW + wave; item < items; item += gridDim.y * (NW / of)) {
        const int which = item & 1, head = (item >> 1) % p.kv_heads, run = (item >> 1) / p.kv_heads;
        const int leader = __builtin_ctzll(__builtin_amdgcn_ballot_w64(leads && rank == run));
        const int64_t t0 = w0 + leader;
        const int64_t s0 = __shfl(slot, leader);
        const int o = (int)(s0 & (ps - 1));
        const int64_t page = s0 >> log2_page;
        // tokens of the run: of these 64, and behind them
        const int place = lane - leader;
        const uint64_t others = ~__builtin_amdgcn_ballot_w64(place >= 0 && place < ps - o && slot == s0 + place) >> leader;
        int n = others ? __builtin_ctzll(others) : 64 - leader;
        while (leader + n >= 64) {
            const int i = n + lane;
            const bool in = i < ps - o && t0 + i < p.tokens && p.slots[t0 + i] == s0 + i;
            const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
            if (mask != ~0ull) {
                n += __builtin_ctzll(~mask);
                break;
            }
            n += 64;
        }

        const float *scale = which ? p.cache.v_scale + page * (p.cache.vs_sp / 4) + head * p.cache.vs_sh
                                   : p.cache.k_scale + page * (p.cache.ks_sp / 4) + head * p.cache.ks_sh;
        const float held = *scale;                // on the way with the rows
        const int64_t st = which ? p.v_st : p.k_st;
        const T *x = which ? (const T *)p.v + t0 * p.v_st + head * p.v_sh : (const T *)p.k + t0 * p.k_st + head * p.k_sh;
        // The new scale, and what it is of.
        float was = 0.f, now = 0.f;
        bool grown = false;
        const auto rescale = [&](float a) {
            a = wave_max(a);
            was = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(held)));
            if (together) {
                if (lane == 0) largest[turn][wave] = a;
                __syncthreads();                  // (and every wave has the old scale)
#pragma unroll
                for (int w = 0; w < NW; ++w) a = fmaxf(a, largest[turn][w]);
                turn ^= 1;
            }
            const float need = cache_scale_for(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(a))));
            const bool kept = o > 0 && was > 0.f && was < INFINITY;
            now = kept ? fmaxf(was, need) : need;
            grown = kept && now != was;
            if (lane == 0 && sub == 0 && !(kept && now == was)) *const_cast<float *>(scale) = now;
        };
        typedef CacheRaw<T, E> Row;
        constexpr int RPI = 64 / LPR;             // rows at a time
        const T *at = x + lane % LPR * E;
        const auto row_at = [&](int i) {           // past the last: the last
            Row r;
            r.load(at + min(i, n - 1) * st);
            return r;
        };
        if (which == 0) {
            uint8_t *k = p.cache.k + page * p.cache.k_sp + head * p.cache.k_sh;
            const auto store = [&](const Row &raw, int i, const auto &quotient) {
                const auto r = raw.get();
                CacheVec<uint32_t, E / 4> c;
#pragma unroll
                for (int j = 0; j < E / 4; ++j) {
                    int q = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r.v[4 * j]), quotient((float)r.v[4 * j + 1]), 0, false);
                    c.v[j] = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r.v[4 * j + 2]), quotient((float)r.v[4 * j + 3]), q, true);
                }
                if (i < n) *(CacheVec<uint32_t, E / 4> *)(k + (int64_t)(o + i) * p.cache.k_st + lane % LPR * E) = c;
            };
            const int first = lane / LPR;
            float a = 0.f;
            Row r[kAppendRows] = {};
            // (a run of a few rows, the usual one of a decoding step, is one vector)
            const bool few = n <= RPI, fits = n <= of * kAppendRows * RPI;
            if (few) {
                r[0] = row_at(first);
                a = finite_max(r[0].get(), a);
            } else {
                for (int i = first + sub * kAppendRows * RPI; i < n; i += of * kAppendRows * RPI) {
#pragma unroll
                    for (int j = 0; j < kAppendRows; ++j) r[j] = row_at(i + j * RPI);
#pragma unroll
                    for (int j = 0; j < kAppendRows; ++j) {
                        a = finite_max(r[j].get(), a);
                        __builtin_amdgcn_sched_barrier(0);   // a row's fp32 values at a time
                    }
                }
            }
            rescale(a);
#pragma unroll
            for (int j = 0; j < kAppendRows; ++j)
                if (j == 0 || !few) r[j].settle();
            with_quotient(now, [&](const auto &quotient) {
                if (few) {
                    if (sub == 0) store(r[0], first, quotient);
                    return;
                }
                for (int i = first + sub * kAppendRows * RPI; i < n; i += of * kAppendRows * RPI) {
                    if (!fits)
#pragma unroll
                        for (int j = 0; j < kAppendRows; ++j) r[j] = row_at(i + j * RPI);
#pragma unroll
                    for (int j = 0; j < kAppendRows; ++j) {
                        store(r[j], i + j * RPI, quotient);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            });
            if (grown) {
                const float shrink = was / now;
                for (int i = sub * (64 / (D / 4)) + lane / (D / 4); i < o; i += of * (64 / (D / 4))) {
                    uint32_t *c = (uint32_t *)(k + (int64_t)i * p.cache.k_st + lane % (D / 4) * 4);
                    *c = cache_rescale(*c, shrink);
                }
            }
        } else {
            uint8_t *v = p.cache.v + page * p.cache.v_sp + head * p.cache.v_sh;
            constexpr int LPC = D / 2;            // lanes that cover the columns, two each
            const int d = lane % LPC * 2;
            typedef CacheRaw<T, 2> Pair;
            typedef CacheVec<uint32_t, 4> Codes;
            // 16 tokens of a page from 16 g on; those outside the run: one of its own, not used
            Pair r[16] = {};
            const auto read = [&](int g) {
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i].load(x + min(max(g * 16 + i - o, 0), n - 1) * st + d);
            };
            const int g0 = o / 16, g1 = (o + n + 15) / 16;
            const bool fits = g1 - g0 == 1;
            Codes a0, a1;
            uint8_t *c0 = v + (int64_t)d * p.cache.v_sd + g0 * 16, *c1 = c0 + p.cache.v_sd;
            float a = 0.f;
            if (fits) {
                a0 = *(Codes *)c0, a1 = *(Codes *)c1;
                read(g0);
#pragma unroll
                for (int i = 0; i < 16; ++i) a = finite_max(r[i].get(), a);
            } else {
                for (int i = sub * 4 * RPI + lane / LPR; i < n; i += of * 4 * RPI) {
                    Row y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = row_at(i + j * RPI);
#pragma unroll
                    for (int j = 0; j < 4; ++j) a = finite_max(y[j].get(), a);
                }
            }
            rescale(a);
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i].settle();
            const float shrink = was / now;
            const bool again = !fits || grown;
            with_quotient(now, [&](const auto &quotient) {
                // (a group at hand is every wave's)
                for (int g = (grown ? 0 : g0) + (again ? sub * (64 / LPC) + lane / LPC : sub); g < g1; g += again ? of * (64 / LPC) : of) {
                    if (again) {
                        c0 = v + (int64_t)d * p.cache.v_sd + g * 16, c1 = c0 + p.cache.v_sd;
                        a0 = *(Codes *)c0, a1 = *(Codes *)c1;
                        read(g);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = g * 16 + 4 * j;
                        const uint32_t fresh = byte_mask(at, o, o + n), old = byte_mask(at, 0, o);
                        const auto pack = [&](int c) -> uint32_t {
                            int q = __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r[4 * j].get().v[c]), quotient((float)r[4 * j + 1].get().v[c]), 0, false);
                            return __builtin_amdgcn_cvt_pk_fp8_f32(quotient((float)r[4 * j + 2].get().v[c]), quotient((float)r[4 * j + 3].get().v[c]), q, true);
                        };
                        if (grown) {
                            a0.v[j] = (cache_rescale(a0.v[j], shrink) & old) | (a0.v[j] & ~old);
                            a1.v[j] = (cache_rescale(a1.v[j], shrink) & old) | (a1.v[j] & ~old);
                        }
                        a0.v[j] = (pack(0) & fresh) | (a0.v[j] & ~fresh);
                        a1.v[j] = (pack(1) & fresh) | (a1.v[j] & ~fresh);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    *(Codes *)c0 = a0;
                    *(Codes *)c1 = a1;
                }
            });
        }
    }
}

}  // namespace pmkl_amd
