// gfx950 attention over the paged 8-bit cache (include/pmkl_cache.h).
//
// The unit of work is a tile of 64 keys for 16 query rows of one request and key
// head: row r is query head r % G of the head's G, token r / G, so that a key is
// read once for all heads that share it.  A wave takes tiles one after the
// other, with a running max, sum and output.  Which wave has which tiles, and
// where they are joined: cache_attn_kernel, cache_split and cache_chunk below.
//
// Scores are formed transposed, S^T = K Q^T, and so is the output, O^T = V^T P^T,
// with v_mfma_f32_16x16x32: codes become exact 16-bit values on the way from the
// load to the matrix unit, two in an instruction.
//   * Of the four 16-key products of a tile, number t has key 16 (i / 4) + 4 t +
//     i % 4 in row i.  Of the results a lane has rows 4 g .. 4 g + 3 (g = lane /
//     16), so over the four it has the 16 consecutive keys 16 g ..: one page's, so
//     one scale of the lane; and they are, in order, the lane's part of the P V
//     product, whose V^T operand is 16 bytes of a column's tokens.  Nothing
//     passes through the LDS or between lanes but the row max.
//   * The contraction over columns may take them in any order, so a lane loads
//     16 consecutive bytes of a key, two operands' worth.
//   * The next tile's keys are loaded when the scores have taken the registers
//     of this one's, its values after P V, its table entries a tile earlier: 16
//     KB (head_dim 128) of a wave are under way at any time.
// Types.  Keys meet bf16 and fp32 queries in bf16 (the latter as three terms, 24
// bits), f16 queries in f16.  P V is in f16: a weight times its page's scale, s, is
// held as p s 2^(14 - E), with the exponent of the tile's largest scale as E, and
// 2^(E - 14) goes into the factor that rescales the output anyway.  That is one f16
// term under bf16 queries (error 2^-12 of a weight, beside the output's 2^-9) and
// two under the others (2^-22), in full while the scales of a tile lie within 2^8
// and p is above 2^-20 (below, 2^-31 is lost); a tile whose scales lie further apart
// takes another round for the larger ones.
#pragma once

#include "cache_common.hpp"

namespace pmkl_amd {

typedef __bf16 cbf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 cf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 cbf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 cf16x8_t __attribute__((ext_vector_type(8)));
typedef float cf32x4_t __attribute__((ext_vector_type(4)));

struct CacheUnfinished;

struct CacheAttnParams {
    const void *q;
    void *o;
    float *m;
    float *l;
    CacheParams cache;
    const int32_t *table;
    const int32_t *seq_lens;
    const int32_t *query_start;
    float *parts;
    CacheUnfinished *unfinished;
    int64_t q_st, q_sh, o_st, o_sh;   // elements
    int64_t table_stride;
    int32_t tokens;
    int32_t batch;
    int32_t width;
    int32_t kv_heads;
    int32_t group;                    // query heads of a key head
    int32_t is_causal;
    float scale;
    int32_t ranges;                   // of the split form
    int32_t chunks;                   // whether chunks have their own workgroups
};

constexpr int kCacheTile = 64;    // keys
constexpr int kCacheRows = 16;    // query rows of a block
constexpr int kPBits = 14;        // weights are held as p s 2^(14 - E)
constexpr int kSpread = 8;        // scales of a product lie within 2^8

// Queries of a type: the 16-bit type of the score product, how many terms a
// query has there, and a weight in f16.
template <typename T> struct CacheQuery;
template <> struct CacheQuery<__bf16> {
    typedef cbf16x8_t frag;
    static constexpr int QT = 1, PT = 1;
};
template <> struct CacheQuery<_Float16> {
    typedef cf16x8_t frag;
    static constexpr int QT = 1, PT = 2;
};
template <> struct CacheQuery<float> {
    typedef cbf16x8_t frag;
    static constexpr int QT = 3, PT = 2;
};

__device__ __forceinline__ cf32x4_t cache_mfma(cbf16x8_t a, cbf16x8_t b, cf32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ cf32x4_t cache_mfma(cf16x8_t a, cf16x8_t b, cf32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// eight codes as an operand
template <typename F>
__device__ __forceinline__ F cache_frag(uint32_t lo, uint32_t hi) {
    if constexpr (__is_same(F, cbf16x8_t)) {
        const cbf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
        const cbf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
        const cbf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
        const cbf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
        return F{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    } else {
        const cf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
        const cf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
        const cf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
        const cf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
        return F{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
}

// x as N terms of a 16-bit type, each the rounding of what those before leave.
// Where x is a product, all terms must start from its fp32 value: contracted into
// the subtraction and the conversions (v_fma_mix), the first term and the one that
// is subtracted can round to different sides.
template <int N, typename H>
__device__ __forceinline__ void cache_terms(float x, H (&t)[N]) {
    if constexpr (N > 1) asm("" : "+v"(x));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        t[i] = (H)x;
        x -= (float)t[i];
    }
}

__device__ __forceinline__ float cache_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Whether a byte of x is the code of NaN (0x7f, 0xff): the high bit of each.
__device__ __forceinline__ uint32_t cache_nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// 16 codes of a column without those past the first `n`, and 0 for NaN (nans collects where).
__device__ __forceinline__ void cache_clear(uint32_t (&x)[4], int n, uint32_t &nans) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int some = min(max(n - 4 * j, 0), 4);
        x[j] &= some ? 0xffffffffu >> (32 - 8 * some) : 0u;
        const uint32_t bad = cache_nan_bytes(x[j]);
        nans |= bad;
        x[j] &= ~(bad | (bad - (bad >> 7)));
    }
}

// Over the four 16-lane rows, of an integer that is the same in all lanes of a row.
template <typename Op>
__device__ __forceinline__ int cache_over_rows(int x, Op op) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = op((int)r[0], (int)r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(op((int)h[0], (int)h[1]));
}

// of a scale >= 0, -126 at least
__device__ __forceinline__ int cache_exponent(float scale) { return max((int)(__float_as_uint(scale) >> 23 & 0xff), 1) - 127; }

// A request's rows of one key head.
struct CacheItem {
    int b, head, row0;      // row0: the block's first row
    int q0, n;              // the request's first token, its tokens
    int length, keys;       // seq_len, and how many of its tokens the table holds
};

__device__ __forceinline__ CacheItem cache_request(const CacheAttnParams &p, int b) {
    CacheItem it;
    it.b = b, it.head = 0, it.row0 = 0;
    it.q0 = min(max(p.query_start[b], 0), p.tokens);
    it.n = min(max(p.query_start[b + 1], it.q0), p.tokens) - it.q0;
    it.length = max(p.seq_lens[b], 0);
    it.keys = min(it.length, p.width << p.cache.log2_page);   // < 2^31 (checked)
    return it;
}

// keys that the request's token t sees
__device__ __forceinline__ int cache_limit(const CacheAttnParams &p, const CacheItem &it, int t) {
    return p.is_causal ? max(min(it.keys, it.length - it.n + t + 1), 0) : it.keys;
}

__device__ __forceinline__ int64_t cache_rows(const CacheAttnParams &p, const CacheItem &it) {
    return (int64_t)it.n * p.group;
}
__device__ __forceinline__ int cache_blocks(const CacheAttnParams &p, const CacheItem &it) {   // of 16 rows
    return (int)((cache_rows(p, it) + kCacheRows - 1) / kCacheRows);
}
// tiles that a row block of the request counts for: its keys' (one at least, so
// that rows that see nothing are written)
__device__ __forceinline__ int cache_tiles(const CacheItem &it) { return max((it.keys + kCacheTile - 1) / kCacheTile, 1); }

__device__ __forceinline__ void cache_uniform(CacheItem &it) {
    it.b = __builtin_amdgcn_readfirstlane(it.b);
    it.head = __builtin_amdgcn_readfirstlane(it.head);
    it.row0 = __builtin_amdgcn_readfirstlane(it.row0);
    it.q0 = __builtin_amdgcn_readfirstlane(it.q0);
    it.n = __builtin_amdgcn_readfirstlane(it.n);
    it.length = __builtin_amdgcn_readfirstlane(it.length);
    it.keys = __builtin_amdgcn_readfirstlane(it.keys);
}

// Whether request b starts behind its end.  Past such a one the sums below would not
// be bounded by what the host has checked: nothing is looked for there.
__device__ __forceinline__ bool cache_falls(const CacheAttnParams &p, int b) {
    return b < p.batch && p.query_start[b + 1] < p.query_start[b];
}

// Requests in order have weight(request) units each (fewer than 2^31 in all:
// checked); finds the one with unit i, and i counted from its first.  Every wave
// sums by itself, 64 requests at a time.  False past the last unit.
template <typename Weight>
__device__ __forceinline__ bool cache_find(const CacheAttnParams &p, int &i, int lane, CacheItem &it, Weight weight) {
    for (int base = 0; base < p.batch; base += 64) {
        const int b = base + lane;
        if (__builtin_amdgcn_ballot_w64(cache_falls(p, b))) return false;
        const int own = b < p.batch ? weight(cache_request(p, b)) : 0;
        const int end = wave_scan(own);
        const uint64_t mask = __builtin_amdgcn_ballot_w64(i < end);
        if (mask) {
            const int l = __builtin_ctzll(mask);
            i -= __builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(own, l);
            it = cache_request(p, base + l);
            return true;
        }
        i -= __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

// A head's pages.  Strides between pages are below 2^31 (checked): a page's place
// is one multiply-add.
struct CacheHead {
    const uint8_t *k, *v;
    const char *ks, *vs;
    const int32_t *table;   // the request's row
    int last_page;

    __device__ __forceinline__ CacheHead(const CacheAttnParams &p, const CacheItem &it) {
        k = p.cache.k + (int64_t)it.head * p.cache.k_sh;
        v = p.cache.v + (int64_t)it.head * p.cache.v_sh;
        ks = (const char *)(p.cache.k_scale + (int64_t)it.head * p.cache.ks_sh);
        vs = (const char *)(p.cache.v_scale + (int64_t)it.head * p.cache.vs_sh);
        table = p.table + (int64_t)it.b * p.table_stride;
        last_page = (it.keys - 1) >> p.cache.log2_page;
    }
    // table entry of the page of a key
    __device__ __forceinline__ int entry(const CacheAttnParams &p, int key) const {
        return table[(uint32_t)min(key >> p.cache.log2_page, last_page)];
    }
};
__device__ __forceinline__ uint32_t cache_page(const CacheAttnParams &p, int entry) {
    return (uint32_t)entry < (uint32_t)p.cache.pages ? entry : 0;
}
template <typename T>
__device__ __forceinline__ const T *cache_at(const T *base, uint32_t page, uint32_t stride) { return base + (uint64_t)page * stride; }

// A wave's rows: QB blocks of 16, of one request and key head, a column of the
// results each.
template <typename T, int D, int QB>
struct CacheRows {
    using CQ = CacheQuery<T>;
    typedef typename CQ::frag frag;
    static constexpr int QT = CQ::QT, PT = CQ::PT;
    static constexpr int NK = D / 32;          // operands of a key
    static constexpr int NB = D / 16;          // 16-column blocks of the output

    frag q[QB][QT][NK];
    cf32x4_t o[QB][NB];     // sum p v, in units of 2^(unit - 14) (relative to m)
    float m[QB], l[QB];     // m in units of log2; l of this lane's keys
    int limit[QB];          // keys that the lane's row sees
    int first_limit, last_limit;   // that the wave's first and last row see
    int unit, peak;
    uint32_t nans;          // what values() had to clear in tiles for step_any()

    // rows it.row0 + 16 b + column, as operands
    __device__ __forceinline__ void load(const CacheAttnParams &p, const CacheItem &it, int lane) {
        const int g = lane >> 4;
        const int64_t rows = cache_rows(p, it);
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int64_t row = (int64_t)it.row0 + b * kCacheRows + (lane & 15);
            const bool live = row < rows;
            const int token = live ? (int)row / p.group : 0;
            limit[b] = live ? cache_limit(p, it, token) : 0;
            const T *src = (const T *)p.q + (int64_t)(it.q0 + token) * p.q_st + (int64_t)(it.head * p.group + (live ? (int)row % p.group : 0)) * p.q_sh;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const int d = D >= 64 ? k / 2 * 64 + g * 16 + k % 2 * 8 : g * 8;
                struct alignas(16) { T v[8]; } x{};
                if (live) x = *(const decltype(x) *)(src + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (QT == 1) {
                        q[b][0][k][e] = x.v[e];
                    } else {
                        __bf16 t[QT];
                        cache_terms<QT>((float)x.v[e], t);
#pragma unroll
                        for (int i = 0; i < QT; ++i) q[b][i][k][e] = t[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) o[b][i] = cf32x4_t{};
            m[b] = -INFINITY, l[b] = 0.f;
        }
        unit = peak = -126;
        nans = 0;
        first_limit = it.row0 < rows ? cache_limit(p, it, it.row0 / p.group) : 0;
        last_limit = last_key(p, it);
    }
    // keys that the last of the rows sees
    static __device__ __forceinline__ int last_key(const CacheAttnParams &p, const CacheItem &it) {
        const int64_t rows = cache_rows(p, it);
        return it.row0 < rows ? cache_limit(p, it, (int)(min((int64_t)it.row0 + QB * kCacheRows, rows) - 1) / p.group) : 0;
    }

    template <typename K>
    __device__ __forceinline__ void scores(cf32x4_t (&s)[QB][4], K keys) const {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int b = 0; b < QB; ++b) s[b][t] = cf32x4_t{};
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const frag a = keys(t, k);
#pragma unroll
                for (int i = QT - 1; i >= 0; --i)    // the smallest first
#pragma unroll
                    for (int b = 0; b < QB; ++b) s[b][t] = cache_mfma(a, q[b][i][k], s[b][t]);
            }
        }
    }

    // Scores (times c) to weights, times 2^shift, of which `unshift` is the inverse;
    // alpha: what the sums so far are worth now.
    __device__ __forceinline__ void weigh(cf32x4_t (&s)[QB][4], float c, float shift, float unshift, float (&alpha)[QB]) {
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            float mx = s[b][0][0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = cache_max(mx, s[b][e / 4][e % 4]);
            mx = cache_max(m[b], across_rows(mx * c, [](float a, float b) { return cache_max(a, b); }));
            const float ref = mx == -INFINITY ? 0.f : mx;
            alpha[b] = __builtin_amdgcn_exp2f(m[b] - ref);
            m[b] = mx;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[b][e / 4][e % 4], c, shift - ref));
                s[b][e / 4][e % 4] = x;
                sum += x;
            }
            l[b] = l[b] * alpha[b] + sum * unshift;
        }
    }

    // o = o alpha + P V, P being s (MASKED: times the lane's weight, where seen[b] > e)
    template <bool MASKED, typename V>
    __device__ __forceinline__ void add(const cf32x4_t (&s)[QB][4], const float (&alpha)[QB], float weight, int now, const int (&seen)[QB], V values) {
        float rescale[QB];
        bool still = true;
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            rescale[b] = __builtin_amdgcn_ldexpf(alpha[b], unit - now);
            still = still && rescale[b] == 1.f;
        }
        unit = now;
        peak = max(peak, now);
        // after the first tiles the largest score seldom changes
        if (__builtin_amdgcn_ballot_w64(!still) != 0)
#pragma unroll
            for (int b = 0; b < QB; ++b)
#pragma unroll
                for (int i = 0; i < NB; ++i) o[b][i] *= rescale[b];
        // eight of the lane's keys, then the others
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            cf16x8_t ph[QB][PT];
#pragma unroll
            for (int b = 0; b < QB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = s[b][h * 2 + e / 4][e % 4];
                    if constexpr (MASKED) x = h * 8 + e < seen[b] ? x * weight : 0.f;   // (of a page that the row does not see the weight may be anything)
                    _Float16 terms[PT];
                    cache_terms<PT>(x, terms);
#pragma unroll
                    for (int i = 0; i < PT; ++i) ph[b][i][e] = terms[i];
                }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const cf16x8_t a = values(i, h);
#pragma unroll
                for (int j = PT - 1; j >= 0; --j)
#pragma unroll
                    for (int b = 0; b < QB; ++b) o[b][i] = cache_mfma(a, ph[b][j], o[b][i]);
            }
        }
    }

    // A tile that every row sees whole, of pages of the cache whose scales lie
    // within 2^8 (their exponents' largest is `now`): nearly all tiles.  keys(t, k)
    // and values(i, h) give the operands; taken() is called when the keys have
    // been taken.
    template <typename K, typename V, typename F>
    __device__ __forceinline__ void step(float c, float vs, int now, K keys, V values, F taken) {
        cf32x4_t s[QB][4];
        float alpha[QB];
        scores(s, keys);
        taken();
        // the values' scale, a factor of the lane, goes into the exponent
        const float weight = __builtin_amdgcn_ldexpf(vs, kPBits - now);
        weigh(s, c, __builtin_amdgcn_logf(weight), __builtin_amdgcn_rcpf(weight), alpha);
        add<false>(s, alpha, 1.f, now, limit, values);
    }

    // Any other tile; its lane has keys vkey .. vkey + 15, `held` if their page is
    // one of the cache's.  values() gives 0 for NaN, and for what no row sees;
    // anew() keeps what they give from being held over the rounds (64 registers).
    template <typename K, typename V, typename F>
    __device__ __forceinline__ void step_any(int vkey, bool held, float c, float vs, K keys, V values, F anew) {
        cf32x4_t s[QB][4];
        float alpha[QB];
        int seen[QB];                                      // of the lane's 16 keys, those below are visible
        scores(s, keys);
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            seen[b] = held ? limit[b] - vkey : 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = s[b][e / 4][e % 4] * c;
                s[b][e / 4][e % 4] = e < seen[b] ? x : -INFINITY;
            }
        }
        weigh(s, 1.f, 0.f, 1.f, alpha);
        // Pages within 2^8 of the least scale take part together, then the others.
        const float scale = held ? vs : 0.f;
        const int exponent = cache_exponent(scale);
        bool todo = held;
        while (__builtin_amdgcn_ballot_w64(todo) != 0) {    // (no page: alpha is 1, or there is nothing yet)
            anew();
            const int least = cache_over_rows(todo ? exponent : 128, [](int a, int b) { return min(a, b); });
            const bool use = todo && exponent <= least + kSpread;
            // (what is summed must not overflow: the unit stays within 2^80 of its highest)
            const int now = max(cache_over_rows(use ? exponent : -126, [](int a, int b) { return max(a, b); }), peak - 80);
            add<true>(s, alpha, use ? __builtin_amdgcn_ldexpf(scale, kPBits - now) : 0.f, now, seen, values);
            todo = todo && !use;
#pragma unroll
            for (int b = 0; b < QB; ++b) alpha[b] = 1.f;
        }
    }

    // Whether step() does for a tile, and its largest exponent.
    __device__ __forceinline__ bool whole(int key0, bool held, float scale, int &now) const {
        const int exponent = cache_exponent(scale);
        now = cache_over_rows(exponent, [](int a, int b) { return max(a, b); });
        return key0 + kCacheTile <= first_limit && now >= peak - 80 &&
               __builtin_amdgcn_ballot_w64(!(held && scale >= 0x1p-126f && exponent >= now - kSpread)) == 0;
    }

    // After the last tile: o in units of 1, l of the row, and NaN to the outputs of
    // the rows that see a NaN value of step_any()'s tiles: tile, tile + step, ... below
    // end.
    __device__ __forceinline__ void finish(const CacheAttnParams &p, const CacheItem &it, int tile, int end, int step, int lane) {
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            l[b] = across_rows(l[b], [](float a, float b) { return a + b; });
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][i][e] = __builtin_amdgcn_ldexpf(o[b][i][e], unit - kPBits);
        }
        if (__builtin_amdgcn_ballot_w64(nans != 0) == 0) return;
        const int g = lane >> 4, r16 = lane & 15, in_page = (1 << p.cache.log2_page) - 1;
        const CacheHead head(p, it);
        for (; tile < end; tile += step) {
            const int vkey = tile * kCacheTile + g * 16;
            const int entry = head.entry(p, vkey);
            const bool held = (uint32_t)entry < (uint32_t)p.cache.pages && vkey < it.keys;
            const uint8_t *vp = cache_at(head.v, held ? entry : 0, p.cache.v_sp) + (vkey & in_page) + (int64_t)r16 * p.cache.v_sd;
            // bf16 ones where a value is NaN, and where a row sees its token
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            words see[QB][2];
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                const int seen = held ? limit[b] - vkey : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) see[b][j / 4][j % 4] = (seen > 2 * j ? 0x3f80u : 0u) | (seen > 2 * j + 1 ? 0x3f800000u : 0u);
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint4 x = *(const uint4 *)(vp + (int64_t)i * 16 * p.cache.v_sd);
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
                words bad[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t f = cache_nan_bytes(v[j]) >> 7;
                    bad[j / 2][j % 2 * 2] = (f & 1 | (f & 0x100) << 8) * 0x3f80u;
                    bad[j / 2][j % 2 * 2 + 1] = (f >> 16 & 1 | (f & 0x1000000) >> 8) * 0x3f80u;
                }
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    cf32x4_t hit{};
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        hit = cache_mfma(__builtin_bit_cast(cbf16x8_t, bad[h]), __builtin_bit_cast(cbf16x8_t, see[b][h]), hit);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hit[e] > 0.f) o[b][i][e] = __builtin_nanf("");
                }
            }
        }
    }
};

// NT: past the caches' usual policy (nontemporal), for tiles that are read once. On
// 1 GiB of scattered 2 KB pages, read by 512 workgroups, 6.7 TB/s against 5.9; but
// chunks whose 32 row blocks share the tiles 670 us against 423.
template <bool NT, typename V>
__device__ __forceinline__ V cache_load(const uint8_t *p) {
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(V) / 4)));
    return __builtin_bit_cast(V, NT ? __builtin_nontemporal_load((const words *)p) : *(const words *)p);
}

// 16 rows whose tiles the wave loads into registers.
template <typename T, int D>
struct CacheWave : CacheRows<T, D, 1> {
    using Rows = CacheRows<T, D, 1>;
    static constexpr int NK = Rows::NK, NB = Rows::NB;
    uint32_t kr[4][2 * NK], vr[NB][4];
    float ks, vs;

    // kp, vp: the lane's part of a page (below)
    template <bool NT>
    __device__ __forceinline__ void load_keys(const CacheAttnParams &p, const CacheHead &head, const uint8_t *kp, int tile, int kentry, int ventry) {
        const uint8_t *kt = cache_at(kp, cache_page(p, kentry), p.cache.k_sp) + (tile * kCacheTile & (1 << p.cache.log2_page) - 1) * p.cache.k_st;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (D >= 64) {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const uint4 x = cache_load<NT, uint4>(kt + c * 64);
                    kr[t][4 * c] = x.x, kr[t][4 * c + 1] = x.y, kr[t][4 * c + 2] = x.z, kr[t][4 * c + 3] = x.w;
                }
            } else {
                const uint2 x = cache_load<NT, uint2>(kt);
                kr[t][0] = x.x, kr[t][1] = x.y;
            }
            kt += 4 * p.cache.k_st;
        }
        const uint32_t page = cache_page(p, ventry);
        ks = *(const float *)cache_at(head.ks, page, p.cache.ks_sp);
        vs = *(const float *)cache_at(head.vs, page, p.cache.vs_sp);
    }
    template <bool NT>
    __device__ __forceinline__ void load_values(const CacheAttnParams &p, const uint8_t *vp, int tile, int ventry) {
        vp = cache_at(vp, cache_page(p, ventry), p.cache.v_sp) + (tile * kCacheTile & (1 << p.cache.log2_page) - 1);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint4 x = cache_load<NT, uint4>(vp);
            vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
            vp += 16 * p.cache.v_sd;
        }
    }

    // Tiles tile, tile + step, ... below end.
    __device__ __forceinline__ void run(const CacheAttnParams &p, const CacheItem &it, int tile, int end, int step, int lane) {
        if (cache_blocks(p, it) == 1)
            tiles<true>(p, it, tile, end, step, lane);
        else
            tiles<false>(p, it, tile, end, step, lane);
    }
    template <bool NT>
    __device__ __forceinline__ void tiles(const CacheAttnParams &p, const CacheItem &it, int tile, int end, int step, int lane) {
        const int g = lane >> 4, r16 = lane & 15, in_page = (1 << p.cache.log2_page) - 1;
        end = min(end, (this->last_key(p, it) + kCacheTile - 1) / kCacheTile);
        if (tile >= end) {
            this->load(p, it, lane);
            return;
        }
        const CacheHead head(p, it);
        // key 16 (r16 / 4) + r16 % 4 of a tile, columns 16 g ..; column r16, key 16 g
        const uint8_t *kp = head.k + (int64_t)((r16 >> 2) * 16 & in_page) * p.cache.k_st + (r16 & 3) * p.cache.k_st + g * (D >= 64 ? 16 : 8);
        const uint8_t *vp = head.v + (g * 16 & in_page) + (int64_t)r16 * p.cache.v_sd;
        const auto entry = [&](int tile, int block) { return head.entry(p, tile * kCacheTile + block * 16); };
        int kentry = entry(tile, r16 >> 2), ventry = entry(tile, g);
        const int next = min(tile + step, end - 1);
        int knext = entry(next, r16 >> 2), vnext = entry(next, g);
        this->load(p, it, lane);
        load_keys<NT>(p, head, kp, tile, kentry, ventry);
        load_values<NT>(p, vp, tile, ventry);
        const float c0 = p.scale * 1.44269504088896341f;
        const auto keys = [&](int t, int k) { return cache_frag<typename Rows::frag>(kr[t][2 * k], kr[t][2 * k + 1]); };
        const auto values = [&](int i, int h) { return cache_frag<cf16x8_t>(vr[i][2 * h], vr[i][2 * h + 1]); };
        // Whole tiles as long as there are such, then the others.
        for (; tile < end; tile += step) {
            const int vkey = tile * kCacheTile + g * 16;
            const bool held = (uint32_t)ventry < (uint32_t)p.cache.pages && vkey < it.keys;
            int now;
            if (!this->whole(tile * kCacheTile, held, vs, now)) break;
            const float c = c0 * ks, scale = vs;
            kentry = knext, ventry = vnext;
            // (always loaded, of a tile there is: joining the value with another
            // would wait for the load here)
            const int ahead = min(tile + 2 * step, end - 1);
            knext = entry(ahead, r16 >> 2), vnext = entry(ahead, g);
            const bool more = tile + step < end;
            this->step(c, scale, now, keys, values,
                       [&] { if (more) load_keys<NT>(p, head, kp, tile + step, kentry, ventry); });
            if (more) load_values<NT>(p, vp, tile + step, ventry);
        }
        const int begin = tile;
        if (tile < end)
            for (; tile < end; tile += step) {
                const int vkey = tile * kCacheTile + g * 16;
                const bool held = (uint32_t)ventry < (uint32_t)p.cache.pages && vkey < it.keys;
#pragma unroll
                for (int i = 0; i < NB; ++i) cache_clear(vr[i], held ? this->last_limit - vkey : 0, this->nans);
                this->step_any(vkey, held, c0 * ks, vs, keys, values, [&] {
#pragma unroll
                    for (int i = 0; i < NB * 4; ++i) asm volatile("" : "+v"(vr[i / 4][i % 4]));
                });
                if (tile + step < end) {
                    kentry = knext, ventry = vnext;
                    const int ahead = min(tile + 2 * step, end - 1);
                    knext = entry(ahead, r16 >> 2), vnext = entry(ahead, g);
                    load_keys<NT>(p, head, kp, tile + step, kentry, ventry);
                    load_values<NT>(p, vp, tile + step, ventry);
                }
            }
        this->finish(p, it, begin, end, step, lane);
    }
};

// Where the rows of a block end: outputs, or a part of them in the workspace
// (o [16][D], then m and l [16] each).
template <int D>
constexpr int cache_part_floats() { return kCacheRows * (D + 2); }

template <typename T, int D>
__device__ __forceinline__ void cache_store(const CacheAttnParams &p, const CacheItem &it, int r, int d, cf32x4_t x, float m, float l) {
    constexpr float kLn2 = 0.693147180559945309f;
    const int t = it.q0 + (it.row0 + r) / p.group, h = it.head * p.group + (it.row0 + r) % p.group;
    const float inverse = l == 0.f ? 0.f : 1.f / l;   // nothing seen: 0
    struct alignas(4 * sizeof(T)) { T v[4]; } y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = (T)(x[e] * inverse);
    *(decltype(y) *)((T *)p.o + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + d) = y;
    if (d == 0) {
        const int64_t at = (int64_t)t * p.kv_heads * p.group + h;
        p.m[at] = m * kLn2;
        p.l[at] = l;
    }
}

// The waves' results joined.
template <int D, int NW>
struct CacheJoin {
    float o[NW][kCacheRows][D + 4];
    float m[NW][kCacheRows], l[NW][kCacheRows];

    template <typename T>
    __device__ __forceinline__ void put(const CacheWave<T, D> &w, int wave, int lane) {
        const int g = lane >> 4, r16 = lane & 15;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *(cf32x4_t *)&o[wave][r16][i * 16 + g * 4] = w.o[0][i];
        if (g == 0) {
            m[wave][r16] = w.m[0];
            l[wave][r16] = w.l[0];
        }
    }
    __device__ __forceinline__ cf32x4_t get(int r, int d, float &mx, float &sum) const {
        mx = m[0][r];
#pragma unroll
        for (int w = 1; w < NW; ++w) mx = cache_max(mx, m[w][r]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        sum = 0.f;
        cf32x4_t x{};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(m[w][r] - ref);
            sum += l[w][r] * f;
            x += *(const cf32x4_t *)&o[w][r][d] * f;
        }
        return x;
    }
};

// A workgroup for each row block, whose NW waves split its tiles.  One request of 128
// keys, fp32, 4 heads of 64: 5.3 us, of which a launch is 2.5; the lengths, the table, the
// tiles and the join come one after the other.
// Waves of a SIMD: fp32 at head_dim 128 spills with two, 16 requests of 1,000 keys 21.1
// us, with one 16.2; fp16 spills less, 17.2 and 15.2, but 128 requests 36.6 and 44.8.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, D >= 128 ? (CacheQuery<T>::QT > 1 ? 1 : 2) : 3) void cache_attn_kernel(CacheAttnParams p) {
    __shared__ __attribute__((aligned(16))) CacheJoin<D, NW> join;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    CacheItem it;
    int i = blockIdx.x;
    if (!cache_find(p, i, lane, it, [&](const CacheItem &r) { return cache_blocks(p, r) * p.kv_heads; })) return;
    const int blocks = cache_blocks(p, it);
    it.head = i / blocks;
    it.row0 = i % blocks * kCacheRows;
    cache_uniform(it);
    CacheWave<T, D> w;
    w.run(p, it, wave, INT32_MAX, NW, lane);
    join.put(w, wave, lane);
    __syncthreads();
    for (int j = tid; j < kCacheRows * D / 4; j += NW * 64) {
        const int r = j / (D / 4), d = j % (D / 4) * 4;
        if (it.row0 + r >= cache_rows(p, it)) break;
        float m, l;
        const cf32x4_t x = join.get(r, d, m, l);
        cache_store<T, D>(p, it, r, d, x, m, l);
    }
}

// Where the call has many rows, a request with the rows of a workgroup or more is
// a chunk and has a form of its own (64 requests of 128 rows 82 us, in the split
// form 103; of 64 rows 75 and 67).
constexpr int kChunkBlocks = 1, kChunkWaves = 8;
constexpr int kChunkRows = kCacheRows * kChunkBlocks * kChunkWaves;
__device__ __forceinline__ bool cache_is_chunk(const CacheAttnParams &p, const CacheItem &r) { return cache_rows(p, r) >= kChunkRows; }

// The tiles of all row blocks, one after the other (requests, then heads, then
// blocks), in equal ranges of a wave each, however the requests' lengths differ:
// the host need not know them.  A block counts for kBlockCost tiles more than it
// has, about what its start and end take a wave; they lie before its first.  A
// block in several ranges leaves a part for each in the workspace, which
// cache_attn_join_kernel adds up: part 2 w of range w is the one that starts the
// range, 2 w + 1 one that starts behind it.  `unfinished` tells the join of the
// block whose first tile is in range w and whose last is not.
// Bound by the cache's bytes where they are many: 128 requests of 512 to 16,384
// tokens, 32 heads over 8 of 128, 1.05 GB in 173 us, 6.1 TB/s; by latency where they
// are few: of the 14 us for 4 of 4,096 (34 MB) some 2.5 go into the lengths and the
// range's place, 2 into the first tile's loads, 1 into each tile's arithmetic.
struct CacheUnfinished {
    int rows;         // of the block, 0: there is none
    int q0, head, row0;
    int parts, first; // how many, and the first's number
    int pad[2];
};
constexpr int kBlockCost = 2;

__device__ __forceinline__ int cache_weight(const CacheAttnParams &p, const CacheItem &r) {
    if (p.chunks && cache_is_chunk(p, r)) return 0;
    return cache_blocks(p, r) * p.kv_heads * (cache_tiles(r) + kBlockCost);
}

template <typename T, int D>
__device__ __forceinline__ void cache_split(const CacheAttnParams &p, int range, int ranges) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
    const auto weight = [&](int b) { return b < p.batch ? cache_weight(p, cache_request(p, b)) : 0; };
    // of the first 64 requests, and of all
    const int own = weight(lane), sums = wave_scan(own), first = __builtin_amdgcn_readlane(sums, 63);
    int rest = 0;
    bool falls = cache_falls(p, lane);
    for (int b = 64 + lane; b < p.batch; b += 64) {
        rest += weight(b);
        falls = falls || cache_falls(p, b);
    }
    if (p.batch > 64) rest = __builtin_amdgcn_readlane(wave_scan(rest), 63);
    const int total = __builtin_amdgcn_ballot_w64(falls) ? 0 : first + rest;
    ranges = min(ranges, total);          // none is empty
    const auto begin_of = [&](int r) { return (int)((int64_t)r * total / ranges); };
    const int lo = range < ranges ? begin_of(range) : 0, hi = range < ranges ? begin_of(range + 1) : 0;
    CacheUnfinished left{};
    CacheItem it;
    int i = lo;                           // the place among the request's
    if (lo < hi) {
        if (lo < first) {
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lo < sums));
            i -= __builtin_amdgcn_readlane(sums, l) - __builtin_amdgcn_readlane(own, l);
            it = cache_request(p, l);
        } else {
            cache_find(p, i, lane, it, [&](const CacheItem &r) { return cache_weight(p, r); });
        }
        cache_uniform(it);
    }
    CacheWave<T, D> w;
    for (int at = lo; at < hi;) {
        const int length = cache_tiles(it) + kBlockCost, blocks = cache_blocks(p, it);
        const int block = i / length;
        const int begin = i - block * length, end = min(length, begin + (hi - at));
        const int from = max(begin - kBlockCost, 0), to = end - kBlockCost;
        if (to > 0) {
            it.head = __builtin_amdgcn_readfirstlane(block / blocks);
            it.row0 = __builtin_amdgcn_readfirstlane(block % blocks * kCacheRows);
            const int rows = (int)min(cache_rows(p, it) - it.row0, (int64_t)kCacheRows);
            w.run(p, it, from, to, 1, lane);
            const int number = 2 * range + (at != lo);
            const bool all = from == 0 && end == length;
            if (from == 0 && end < length)
                left = CacheUnfinished{rows, it.q0, it.head, it.row0,
                                       (int)(((int64_t)(at - begin + length) * ranges - 1) / total) - range + 1, number, {0, 0}};
            float *part = p.parts + (int64_t)number * cache_part_floats<D>();
            if (r16 < rows) {
                if (all) {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) cache_store<T, D>(p, it, r16, j * 16 + g * 4, w.o[0][j], w.m[0], w.l[0]);
                } else {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) *(cf32x4_t *)(part + r16 * D + j * 16 + g * 4) = w.o[0][j];
                    if (g == 0) {
                        part[kCacheRows * D + r16] = w.m[0];
                        part[kCacheRows * (D + 1) + r16] = w.l[0];
                    }
                }
            }
        }
        at += end - begin;
        i += end - begin;
        if (at < hi && i >= length * blocks * p.kv_heads) {
            i = 0;
            do it = cache_request(p, it.b + 1);
            while (cache_weight(p, it) == 0);
            cache_uniform(it);
        }
    }
    if (lane == 0) p.unfinished[range] = left;
}

constexpr int kSplitWaves = 4;   // of a workgroup: they share nothing

// Waves that a SIMD holds of the kernel, whose registers are as many as that leaves:
// with fewer they spill (head_dim 128 in two terms, 128 requests of 16 k, us: one wave
// 186 in fp16 and 191 in fp32, two 294 and 340; head_dim 64 in fp16, 64 requests of 4 k:
// two 17.7, three 22.1; head_dim 32 three 27.0, two 30.2).
template <typename T, int D>
__host__ __device__ constexpr int cache_split_waves() {
    return D >= 128 && CacheQuery<T>::PT > 1 ? 1 : D >= 64 ? 2 : 3;
}

template <typename T, int D>
__global__ __launch_bounds__(kSplitWaves * 64, (cache_split_waves<T, D>())) void cache_attn_split_kernel(CacheAttnParams p) {
    cache_split<T, D>(p, blockIdx.x * kSplitWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p.ranges);
}

// Adds up the parts of the blocks that ranges leave unfinished.  A workgroup looks
// at PER ranges and takes their blocks one after the other; a row has NW waves,
// over the rows (a power of two), whose D / 4 lanes have the columns of a part.
// Parts come from the L2s of other dies, 2 us away: a wave has eight on the way at
// once, with what they weigh.  Blocks of more than 64 parts take NW 16, PER 4, blocks of
// a few NW 4, PER 1, others NW 8, PER 2 (the attention with each, us: 128 parts 19.9,
// 28.5, 22.8; 6 parts 36.0, 27.0, 29.5; 25 parts 23.1, 17.7, 18.5 to 22.8, 15.9, 15.4).
template <typename T, int D, int NW, int PER>
__global__ __launch_bounds__(NW * 64) void cache_attn_join_kernel(CacheAttnParams p) {
    __shared__ __attribute__((aligned(16))) float share[NW][D];
    __shared__ float share_m[NW], share_l[NW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int PF = cache_part_floats<D>();
    constexpr int SL = 64 / (D / 4);                                // parts of a load
    const int slice = lane / (D / 4), d = lane % (D / 4) * 4;
    int rows[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) rows[j] = p.unfinished[blockIdx.x * PER + j].rows;
    bool used = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (rows[j] == 0) continue;
        const int range = blockIdx.x * PER + j;
        const CacheUnfinished u = p.unfinished[range];
        CacheItem it;
        it.q0 = u.q0, it.head = u.head, it.row0 = u.row0;
        const float *first = p.parts + (int64_t)u.first * PF;
        const float *rest = p.parts + 2 * (int64_t)range * PF;      // part k > 0 is rest[2 k]
        const int waves = max(NW >> (32 - __builtin_clz(u.rows) - ((u.rows & (u.rows - 1)) == 0 ? 1 : 0)), 1);   // of a row
        const int sub = wave % waves;
        if (used) __syncthreads();                                   // the block before has left the LDS
        for (int r = wave / waves; r < (waves > 1 ? wave / waves + 1 : u.rows); r += NW / waves) {
            // (several waves have one row each, and meet below; there may be none for it)
            float m = -INFINITY, l = 0.f;
            cf32x4_t x{};
            for (int k0 = sub * SL + slice; r < u.rows && k0 < u.parts; k0 += SL * waves * 8) {
                float pm[8], pl[8];
                cf32x4_t px[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int k = min(k0 + e * SL * waves, u.parts - 1);
                    const float *part = k ? rest + (int64_t)2 * k * PF : first;
                    pm[e] = part[kCacheRows * D + r];
                    pl[e] = part[kCacheRows * (D + 1) + r];
                    px[e] = *(const cf32x4_t *)(part + r * D + d);
                }
                float mx = m;
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = cache_max(mx, pm[e]);
                const float ref = mx == -INFINITY ? 0.f : mx;
                const float f = __builtin_amdgcn_exp2f(m - ref);
                m = mx, l *= f, x *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k0 + e * SL * waves < u.parts) {
                        const float w = __builtin_amdgcn_exp2f(pm[e] - ref);
                        l += pl[e] * w;
                        x += px[e] * w;
                    }
            }
            // over the lanes of a column
            const auto join = [&](float m2, float l2, cf32x4_t x2) {
                const float mx = cache_max(m, m2), ref = mx == -INFINITY ? 0.f : mx;
                const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
                m = mx;
                l = l * f + l2 * f2;
                x = x * f + x2 * f2;
            };
#pragma unroll
            for (int y = D / 4; y < 64; y <<= 1) {
                cf32x4_t x2;
#pragma unroll
                for (int e = 0; e < 4; ++e) x2[e] = __shfl_xor(x[e], y);
                join(__shfl_xor(m, y), __shfl_xor(l, y), x2);
            }
            if (waves > 1) {
                if (slice == 0) *(cf32x4_t *)&share[wave][d] = x;
                if (lane == 0) share_m[wave] = m, share_l[wave] = l;
                __syncthreads();
                used = true;
                if (sub == 0)
                    for (int w = 1; w < waves; ++w) join(share_m[wave + w], share_l[wave + w], *(const cf32x4_t *)&share[wave + w][d]);
            }
            if (sub == 0 && slice == 0 && r < u.rows) cache_store<T, D>(p, it, r, d, x, m, l);
        }
    }
}

// Chunks of prompts: a workgroup has 128 rows, 16 a wave, and all their tiles.  Its
// waves load a tile's codes together, while they work on the one before, and put
// them into the LDS as the operands that the products take: a code is converted
// once for 128 rows.  In the LDS 16-byte pieces change places within a row, by the
// row's number, so that the 16 rows that a read takes lie in all banks.  Bound by
// what goes beside the products (weights, conversions, LDS reads): 4 chunks of 512 tokens
// over 4,096, bf16, 32 heads over 8 of 128, 129 GFLOP in 186 us, 690 TFLOP/s.
template <typename frag, int D>
struct CacheStage {
    static constexpr int KP = D / 16;                       // 16-code pieces of a key (of a column: 4)
    static constexpr int PIECES = kCacheTile * KP;          // of a tile's keys, and of its values
    static constexpr int BYTES = 2 * PIECES * 32;           // of the LDS
    static constexpr int N = PIECES / (kChunkWaves * 64);   // a thread's, of keys and of values; 0: the first PIECES threads have keys, the next values
    static constexpr int M = N > 0 ? N : 1;

    const uint8_t *kat[M], *vat[M];   // the thread's pieces in a page
    int32_t kentry[M], ventry[M];     // the pages that the next ones are in
    uint4 k[M], v[M];

    static __device__ __forceinline__ int piece(int n, int tid) { return N > 0 ? n * kChunkWaves * 64 + tid : tid % PIECES; }
    static __device__ __forceinline__ bool has_keys(int tid) { return N > 0 || tid < PIECES; }
    static __device__ __forceinline__ bool has_values(int tid) { return N > 0 || (tid >= PIECES && tid < 2 * PIECES); }
    // What the pieces' numbers in a row are xored with.  A read of 16 bytes a lane
    // serves 16 lanes at a time, which are rows 0 - 3 and 12 - 15 of one piece and
    // 4 - 11 of the next, or the other way round; these lie in 16 places.
    static __device__ __forceinline__ int swap8(int i) { return i & 4 | (i & 1) << 1 | (i >> 1 ^ i >> 2) & 1; }
    static __device__ __forceinline__ int key_swap(int row) {
        const int a = row >> 4 & 3;
        return D == 128 ? a * 4 + (row & 3) : D == 64 ? swap8(a * 2 + (row >> 1 & 1)) : (a >> 1 ^ a & 1) << 1 | a >> 1;
    }
    static __device__ __forceinline__ int value_swap(int d) { return swap8(d >> 1 & 7); }

    __device__ __forceinline__ void place(const CacheAttnParams &p, const CacheHead &head, int tid) {
        const int in_page = (1 << p.cache.log2_page) - 1;
#pragma unroll
        for (int n = 0; n < M; ++n) {
            const int x = piece(n, tid);
            kat[n] = head.k + (int64_t)(x / KP & in_page) * p.cache.k_st + x % KP * 16;
            vat[n] = head.v + (x % 4 * 16 & in_page) + (int64_t)(x / 4) * p.cache.v_sd;
        }
    }
    __device__ __forceinline__ void look_up(const CacheAttnParams &p, const CacheHead &head, int tile, int tid) {
#pragma unroll
        for (int n = 0; n < M; ++n) {
            const int x = piece(n, tid);
            kentry[n] = head.entry(p, tile * kCacheTile + x / KP);
            ventry[n] = head.entry(p, tile * kCacheTile + x % 4 * 16);
        }
    }
    __device__ __forceinline__ void load(const CacheAttnParams &p, int tile, int tid) {
        const int first = tile * kCacheTile & (1 << p.cache.log2_page) - 1;
#pragma unroll
        for (int n = 0; n < M; ++n) {
            if (has_keys(tid)) k[n] = *(const uint4 *)(cache_at(kat[n], cache_page(p, kentry[n]), p.cache.k_sp) + (uint32_t)(first * p.cache.k_st));
            if (has_values(tid)) v[n] = *(const uint4 *)(cache_at(vat[n], cache_page(p, ventry[n]), p.cache.v_sp) + first);
        }
    }
    // `any`: the tile is for step_any(): values past `limit` or of no page are cleared, and NaN
    __device__ __forceinline__ void store(const CacheAttnParams &p, const CacheItem &it, uint8_t *stage, int tile, int tid, const int32_t (&entry)[M], bool any,
                                          int limit, uint32_t &nans) const {
#pragma unroll
        for (int n = 0; n < M; ++n) {
            const int x = piece(n, tid);
            if (has_keys(tid)) {
                uint8_t *row = stage + x / KP * (D * 2);
                const int at = x % KP * 2, swap = key_swap(x / KP);
                *(frag *)(row + (at ^ swap) * 16) = cache_frag<frag>(k[n].x, k[n].y);
                *(frag *)(row + (at + 1 ^ swap) * 16) = cache_frag<frag>(k[n].z, k[n].w);
            }
            if (has_values(tid)) {
                uint32_t c[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
                if (any) {
                    const int key = tile * kCacheTile + x % 4 * 16;
                    const bool held = (uint32_t)entry[n] < (uint32_t)p.cache.pages && key < it.keys;
                    cache_clear(c, held ? limit - key : 0, nans);
                }
                uint8_t *row = stage + BYTES / 2 + x / 4 * (kCacheTile * 2);
                const int at = x % 4 * 2, swap = value_swap(x / 4);
                *(cf16x8_t *)(row + (at ^ swap) * 16) = cache_frag<cf16x8_t>(c[0], c[1]);
                *(cf16x8_t *)(row + (at + 1 ^ swap) * 16) = cache_frag<cf16x8_t>(c[2], c[3]);
            }
        }
    }
};

// Where a lane reads its operands in a stage.
template <typename frag, int D>
struct CacheTaker {
    using Stage = CacheStage<frag, D>;
    int key_at[D / 32], value_at[2];
    __device__ __forceinline__ explicit CacheTaker(int lane) {
        const int g = lane >> 4, r16 = lane & 15, row = (r16 >> 2) * 16 + (r16 & 3);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const int at = D >= 64 ? k / 2 * 8 + g * 2 + k % 2 : g;
            key_at[k] = row * (D * 2) + (at ^ Stage::key_swap(row)) * 16;     // (4 rows on: the same swap)
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            value_at[h] = Stage::BYTES / 2 + r16 * (kCacheTile * 2) + (g * 2 + h ^ Stage::value_swap(r16)) * 16;
    }
    __device__ __forceinline__ frag key(const uint8_t *stage, int t, int k) const {
        return *(const frag *)(stage + key_at[k] + t * (4 * D * 2));
    }
    __device__ __forceinline__ cf16x8_t value(const uint8_t *stage, int i, int h) const {
        return *(const cf16x8_t *)(stage + value_at[h] + i * (16 * kCacheTile * 2));
    }
};

template <typename T, int D>
__device__ __forceinline__ void cache_chunk(const CacheAttnParams &p, uint8_t *smem, int *bad, int i) {
    using Rows = CacheRows<T, D, kChunkBlocks>;
    using Stage = CacheStage<typename Rows::frag, D>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const auto blocks = [&](const CacheItem &r) {
        return cache_is_chunk(p, r) ? (int)((cache_rows(p, r) + kChunkRows - 1) / kChunkRows) : 0;
    };
    CacheItem it;
    if (!cache_find(p, i, lane, it, [&](const CacheItem &r) { return blocks(r) * p.kv_heads; })) return;
    const int n = blocks(it);
    // The rows that see the most first (a whole prompt of 8,192 tokens 645 us, in
    // rows' order 970), and for each the heads, so that dies have heads of their own.
    it.head = i % p.kv_heads;
    const int row0 = __builtin_amdgcn_readfirstlane((n - 1 - i / p.kv_heads) * kChunkRows);
    it.row0 = row0 + wave * kChunkBlocks * kCacheRows;
    cache_uniform(it);
    const int64_t rows = cache_rows(p, it);
    // what the workgroup's last and first row see: waves take the same tiles as whole
    const int last = cache_limit(p, it, (int)(min((int64_t)row0 + kChunkRows, rows) - 1) / p.group);
    const int tiles = (last + kCacheTile - 1) / kCacheTile;

    int any = 0;
    Rows w;
    w.load(p, it, lane);
    w.first_limit = cache_limit(p, it, row0 / p.group);
    if (tid == 0) *bad = 0;
    if (tiles > 0) {
        const CacheHead head(p, it);
        const auto entry = [&](int tile) { return head.entry(p, tile * kCacheTile + g * 16); };
        const float c0 = p.scale * 1.44269504088896341f;
        Stage stage;
        uint32_t nans = 0;
        stage.place(p, head, tid);
        stage.look_up(p, head, 0, tid);
        int lane_entry = entry(0);
        stage.load(p, 0, tid);
        float ks, vs;
        bool held;
        int largest;
        // the lane's scales of a tile, and whether step() does for it
        const auto inspect = [&](int tile) {
            const uint32_t page = cache_page(p, lane_entry);
            ks = *(const float *)cache_at(head.ks, page, p.cache.ks_sp);
            vs = *(const float *)cache_at(head.vs, page, p.cache.vs_sp);
            held = (uint32_t)lane_entry < (uint32_t)p.cache.pages && tile * kCacheTile + g * 16 < it.keys;
        };
        inspect(0);
        int32_t ventry[Stage::M];
#pragma unroll
        for (int j = 0; j < Stage::M; ++j) ventry[j] = stage.ventry[j];
        int ahead = min(1, tiles - 1);
        stage.look_up(p, head, ahead, tid);
        lane_entry = entry(ahead);
        bool whole = w.whole(0, held, vs, largest);
        stage.store(p, it, smem, 0, tid, ventry, !whole, last, nans);
        int tile = 0;
        // the workgroup's share in the next tile's stage, before and after a tile's products
        const auto before = [&] {
            __syncthreads();    // the tile is there, and the other half is free
            if (tile + 1 < tiles) stage.load(p, tile + 1, tid);
#pragma unroll
            for (int j = 0; j < Stage::M; ++j) ventry[j] = stage.ventry[j];
            inspect(min(tile + 1, tiles - 1));
            ahead = min(tile + 2, tiles - 1);
            stage.look_up(p, head, ahead, tid);
            lane_entry = entry(ahead);
        };
        const auto after = [&] {
            if (tile + 1 < tiles) {
                whole = whole && w.whole((tile + 1) * kCacheTile, held, vs, largest);
                stage.store(p, it, smem + (tile + 1 & 1) * Stage::BYTES, tile + 1, tid, ventry, !whole, last, nans);
            }
        };
        const CacheTaker<typename Rows::frag, D> taker(lane);
        const auto keys = [&](int t, int k) { return taker.key(smem + (tile & 1) * Stage::BYTES, t, k); };
        const auto values = [&](int i, int h) { return taker.value(smem + (tile & 1) * Stage::BYTES, i, h); };
        // Whole tiles as long as there are such, then the others.
        for (; tile < tiles && whole; ++tile) {
            const float c = c0 * ks, scale = vs;
            const int now = largest;
            before();
            w.step(c, scale, now, keys, values, [] {});
            after();
        }
        const int begin = tile;
        for (; tile < tiles; ++tile) {
            const float c = c0 * ks, scale = vs;
            const bool here = held;
            before();
            if (tile * kCacheTile < w.last_limit)
                w.step_any(tile * kCacheTile + g * 16, here, c, scale, keys, values, [] { asm volatile("" ::: "memory"); });
            after();
        }
        if (nans) *bad = 1;
        __syncthreads();
        w.nans = *bad;
        any = begin;
    }
    if (it.row0 >= rows) return;
    w.finish(p, it, any, (w.last_limit + kCacheTile - 1) / kCacheTile, 1, lane);
#pragma unroll
    for (int b = 0; b < kChunkBlocks; ++b) {
        const int r = b * kCacheRows + (lane & 15);
        if (it.row0 + r < rows) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) cache_store<T, D>(p, it, r, i * 16 + g * 4, w.o[b][i], w.m[b], w.l[b]);
        }
    }
}

// Two workgroups of a CU; one where three terms of a query of 128 columns would spill
// (fp32, a prompt of 8,192 tokens: 725 us, with two 924).
template <typename T, int D>
__global__ __launch_bounds__(kChunkWaves * 64, kChunkWaves / 4 * (D >= 128 && CacheQuery<T>::QT > 1 ? 1 : 2)) void cache_attn_chunk_kernel(CacheAttnParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * CacheStage<typename CacheQuery<T>::frag, D>::BYTES];
    __shared__ int bad;
    cache_chunk<T, D>(p, smem, &bad, blockIdx.x);
}

}  // namespace pmkl_amd
