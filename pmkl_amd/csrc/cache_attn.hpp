// gfx950 attention over the paged 8-bit cache (include/pmkl_cache.h).
//
// A workgroup owns 16 query rows of one request and key head: row r is query
// head r % G of the head's G, token r / G, so that a key is read once for all
// heads that share it.  Its waves take the request's tiles of 64 tokens in turn,
// each with a running max, sum and output of its own, which the LDS joins at the
// end.
//
// Scores are formed transposed, S^T = K Q^T, and so is the output, O^T = V^T P^T,
// with v_mfma_f32_16x16x32: codes become exact bf16 (f16 under f16 queries) on
// the way from the load to the matrix unit, two in an instruction, and the
// page's scale is a factor of the scores or probabilities.
//   * Tile t of the four 16-key tiles has key 16 (i / 4) + 4 t + i % 4 in row i.
//     Of the result a lane has rows 4 g .. 4 g + 3 (g = lane / 16), so over the
//     four tiles it has the 16 consecutive keys 16 g ..: one page's, so one scale
//     of the lane; and they are, in order, the lane's part of the P V product,
//     whose V^T operand is 16 bytes of a column's tokens.  Nothing passes
//     through the LDS or between lanes but the row max.
//   * The contraction over columns may take them in any order, so a lane loads
//     16 consecutive bytes of a key, two operands' worth.
// fp32 queries are three bf16 terms (24 bits).  P is two bf16 terms, error 2^-17
// (three under fp32 queries): with one, its 2^-9 would be as large as the
// rounding of a bf16 output.
#pragma once

#include "cache_common.hpp"

namespace pmkl_amd {

typedef __bf16 cbf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 cf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 cbf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 cf16x8_t __attribute__((ext_vector_type(8)));
typedef float cf32x4_t __attribute__((ext_vector_type(4)));

struct CacheAttnParams {
    const void *q;
    void *o;
    float *m;
    float *l;
    CacheParams cache;
    const int32_t *table;
    const int32_t *seq_lens;
    const int32_t *query_start;
    int64_t q_st, q_sh, o_st, o_sh;   // elements
    int64_t table_stride;
    int32_t tokens;
    int32_t batch;
    int32_t width;
    int32_t kv_heads;
    int32_t group;                    // query heads of a key head
    int32_t is_causal;
    float scale;
};

constexpr int kCacheTile = 64;   // keys

// Queries of a type: how many terms, and the 16-bit type of the score product.
template <typename T> struct CacheQuery;
template <> struct CacheQuery<__bf16> {
    typedef cbf16x8_t frag;
    static constexpr int QT = 1, PT = 2;
};
template <> struct CacheQuery<_Float16> {
    typedef cf16x8_t frag;
    static constexpr int QT = 1, PT = 2;
};
template <> struct CacheQuery<float> {
    typedef cbf16x8_t frag;
    static constexpr int QT = 3, PT = 3;
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

// x as N bf16 terms, each the rounding of what those before leave
template <int N>
__device__ __forceinline__ void cache_terms(float x, __bf16 (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        t[i] = (__bf16)x;
        x -= (float)t[i];
    }
}

__device__ __forceinline__ float cache_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Whether a byte of x is the code of NaN (0x7f, 0xff): the high bit of each.
__device__ __forceinline__ uint32_t cache_nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A workgroup's rows.
struct CacheItem {
    int b, head, row0;      // row0: first row of the tile, rows are token * group + head in the group
    int q0, n;              // the request's first token, its tokens
    int length, keys;       // seq_len, and how many of its tokens the table holds
};

__device__ __forceinline__ CacheItem cache_request(const CacheAttnParams &p, int b) {
    CacheItem it;
    it.b = b;
    it.q0 = min(max(p.query_start[b], 0), p.tokens);
    it.n = min(max(p.query_start[b + 1], it.q0), p.tokens) - it.q0;
    it.length = max(p.seq_lens[b], 0);
    it.keys = (int)min((int64_t)it.length, (int64_t)p.width << p.cache.log2_page);
    return it;
}

// keys that row t of the request's tokens sees
__device__ __forceinline__ int cache_limit(const CacheAttnParams &p, const CacheItem &it, int t) {
    return p.is_causal ? max(min(it.keys, it.length - it.n + t + 1), 0) : it.keys;
}

// The request and rows of work item i (tiles of R rows, then heads, then
// requests): each wave sums the requests' tiles by itself.  False past the last.
template <int R>
__device__ __forceinline__ bool cache_find(const CacheAttnParams &p, int64_t i, int lane, CacheItem &it) {
    int64_t sum = 0;
    for (int base = 0; base < p.batch; base += 64) {
        const int b = base + lane;
        int64_t tiles = 0;
        if (b < p.batch) {
            const CacheItem r = cache_request(p, b);
            tiles = ((int64_t)r.n * p.group + R - 1) / R * p.kv_heads;
        }
        const int64_t end = wave_scan(tiles, lane) + sum;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(i < end);
        if (mask) {
            const int l = __builtin_ctzll(mask);
            it = cache_request(p, base + l);
            const int64_t rem = i - (__shfl(end, l) - __shfl(tiles, l));
            const int per_head = (int)(__shfl(tiles, l) / p.kv_heads);
            it.head = (int)(rem / per_head);
            it.row0 = (int)(rem % per_head) * R;
            return true;
        }
        sum = __shfl(end, 63);
    }
    return false;
}

// NW waves; 16 rows of the workgroup.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void cache_attn_kernel(CacheAttnParams p) {
    using CQ = CacheQuery<T>;
    typedef typename CQ::frag frag;
    constexpr int QT = CQ::QT, PT = CQ::PT;
    constexpr int R = 16;
    constexpr int NK = D / 32;          // operands of a key
    constexpr int NB = D / 16;          // 16-column blocks of the output
    constexpr int LD = D + 4;           // row of the LDS
    constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
    __shared__ __attribute__((aligned(16))) float part[NW][R][LD];
    __shared__ float part_m[NW][R], part_l[NW][R];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r16 = lane & 15;
    CacheItem it;
    if (!cache_find<R>(p, blockIdx.x, lane, it)) return;
    it.b = __builtin_amdgcn_readfirstlane(it.b);
    it.head = __builtin_amdgcn_readfirstlane(it.head);
    it.row0 = __builtin_amdgcn_readfirstlane(it.row0);
    it.q0 = __builtin_amdgcn_readfirstlane(it.q0);
    it.n = __builtin_amdgcn_readfirstlane(it.n);
    it.length = __builtin_amdgcn_readfirstlane(it.length);
    it.keys = __builtin_amdgcn_readfirstlane(it.keys);
    const int64_t rows = (int64_t)it.n * p.group;   // < 2^31 (checked)

    // this lane's row, and its query as operands
    const int row = it.row0 + r16;
    const bool live = row < rows;
    const int token = live ? row / p.group : 0;
    const int limit = live ? cache_limit(p, it, token) : 0;
    frag q[QT][NK];
    {
        const T *src = (const T *)p.q + (int64_t)(it.q0 + token) * p.q_st + (int64_t)(it.head * p.group + (live ? row % p.group : 0)) * p.q_sh;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = D >= 64 ? k / 2 * 64 + g * 16 + k % 2 * 8 : g * 8;
            struct alignas(16) { T v[8]; } x{};
            if (live) x = *(const decltype(x) *)(src + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (QT == 1) {
                    q[0][k][e] = x.v[e];
                } else {
                    __bf16 t[QT];
                    cache_terms<QT>((float)x.v[e], t);
#pragma unroll
                    for (int i = 0; i < QT; ++i) q[i][k][e] = t[i];
                }
            }
        }
    }
    // what the tile's first and last row see
    const int first_limit = cache_limit(p, it, it.row0 / p.group);
    const int last_limit = cache_limit(p, it, (int)(min((int64_t)it.row0 + R, rows) - 1) / p.group);
    const int tiles = (last_limit + kCacheTile - 1) / kCacheTile;

    const uint8_t *kbase = p.cache.k + (int64_t)it.head * p.cache.k_sh;
    const uint8_t *vbase = p.cache.v + (int64_t)it.head * p.cache.v_sh;
    const float *ksbase = p.cache.k_scale + (int64_t)it.head * p.cache.ks_sh;
    const float *vsbase = p.cache.v_scale + (int64_t)it.head * p.cache.vs_sh;
    const int32_t *table = p.table + (int64_t)it.b * p.table_stride;
    const int in_page = (1 << p.cache.log2_page) - 1;
    const float c0 = p.scale * kLog2e;

    cf32x4_t o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = cf32x4_t{};
    float m = -INFINITY, l = 0.f;       // in units of log2; l of this lane's keys

    for (int tile = wave; tile < tiles; tile += NW) {
        const int key0 = tile * kCacheTile;
        // the page of the rows that the lane loads, and of the keys it owns
        const int kkey = key0 + (r16 >> 2) * 16, vkey = key0 + g * 16;
        const int last_page = (it.keys - 1) >> p.cache.log2_page;
        const int kentry = table[min(kkey >> p.cache.log2_page, last_page)];
        const int ventry = table[min(vkey >> p.cache.log2_page, last_page)];
        const bool held = (uint32_t)ventry < (uint32_t)p.cache.pages && vkey < it.keys;
        const int64_t kpage = (uint32_t)kentry < (uint32_t)p.cache.pages ? kentry : 0;
        const int64_t vpage = (uint32_t)ventry < (uint32_t)p.cache.pages ? ventry : 0;

        const float ks = ksbase[vpage * p.cache.ks_sp], vs = vsbase[vpage * p.cache.vs_sp];
        const uint8_t *kp = kbase + kpage * p.cache.k_sp + (int64_t)((kkey & in_page) + (r16 & 3)) * p.cache.k_st;
        const uint8_t *vp = vbase + vpage * p.cache.v_sp + (vkey & in_page) + (int64_t)r16 * p.cache.v_sd;

        uint32_t kr[4][2 * NK], vr[NB][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t *kt = kp + t * 4 * p.cache.k_st;
            if constexpr (D >= 64) {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const uint4 x = *(const uint4 *)(kt + c * 64 + g * 16);
                    kr[t][4 * c] = x.x, kr[t][4 * c + 1] = x.y, kr[t][4 * c + 2] = x.z, kr[t][4 * c + 3] = x.w;
                }
            } else {
                const uint2 x = *(const uint2 *)(kt + g * 8);
                kr[t][0] = x.x, kr[t][1] = x.y;
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint4 x = *(const uint4 *)(vp + (int64_t)i * 16 * p.cache.v_sd);
            vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
        }

        cf32x4_t s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = cf32x4_t{};
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const frag a = cache_frag<frag>(kr[t][2 * k], kr[t][2 * k + 1]);
#pragma unroll
                for (int i = QT - 1; i >= 0; --i) s[t] = cache_mfma(a, q[i][k], s[t]);   // the smallest first
            }
        }
        const float c = c0 * ks;
        const bool masked = key0 + kCacheTile > first_limit || __builtin_amdgcn_ballot_w64(!held) != 0;
        const int seen = held ? limit - vkey : 0;     // of the lane's 16 keys, those below are visible
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] *= c;
                if (masked && 4 * t + e >= seen) s[t][e] = -INFINITY;
                mx = cache_max(mx, s[t][e]);
            }
        mx = cache_max(m, across_rows(mx, [](float a, float b) { return cache_max(a, b); }));
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        cbf16x8_t ph[PT][2];
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(s[t][e] - ref);
                sum += x;
                float y = x * vs;
                if (masked && 4 * t + e >= seen) y = 0.f;
                __bf16 terms[PT];
                cache_terms<PT>(y, terms);
#pragma unroll
                for (int i = 0; i < PT; ++i) ph[i][t / 2][t % 2 * 4 + e] = terms[i];
            }
        l = l * alpha + sum;
#pragma unroll
        for (int i = 0; i < NB; ++i) o[i] *= alpha;

        if (masked) {
            // Hidden values count for nothing, also where they are NaN: what no
            // row sees is cleared, a NaN that some rows see becomes 0 and is
            // put into these rows' outputs.
            uint32_t nans = 0;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = held ? min(max(last_limit - vkey - 4 * j, 0), 4) : 0;
                    vr[i][j] &= n ? 0xffffffffu >> (32 - 8 * n) : 0u;
                    nans |= cache_nan_bytes(vr[i][j]);
                }
            if (__builtin_amdgcn_ballot_w64(nans != 0)) {
                cbf16x8_t see[2];
#pragma unroll
                for (int e = 0; e < 16; ++e) see[e / 8][e % 8] = (__bf16)(e < seen ? 1.f : 0.f);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    cf32x4_t hit{};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        cbf16x8_t bad;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t f = cache_nan_bytes(vr[i][2 * h + j]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) bad[4 * j + e] = (__bf16)(f >> (8 * e + 7) & 1 ? 1.f : 0.f);
                            vr[i][2 * h + j] &= ~((f >> 7) * 0xffu);
                        }
                        hit = cache_mfma(bad, see[h], hit);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hit[e] > 0.f) o[i][e] = __builtin_nanf("");
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const cbf16x8_t a = cache_frag<cbf16x8_t>(vr[i][2 * h], vr[i][2 * h + 1]);
#pragma unroll
                for (int j = PT - 1; j >= 0; --j) o[i] = cache_mfma(a, ph[j][h], o[i]);
            }
    }

    // Join the waves.
    l = across_rows(l, [](float a, float b) { return a + b; });
#pragma unroll
    for (int i = 0; i < NB; ++i) *(cf32x4_t *)&part[wave][r16][i * 16 + g * 4] = o[i];
    if (g == 0) {
        part_m[wave][r16] = m;
        part_l[wave][r16] = l;
    }
    __syncthreads();
    for (int i = tid; i < R * D / 4; i += NW * 64) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (it.row0 + r >= rows) continue;
        float mx = part_m[0][r];
#pragma unroll
        for (int w = 1; w < NW; ++w) mx = cache_max(mx, part_m[w][r]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
        cf32x4_t x{};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(part_m[w][r] - ref);
            sum += part_l[w][r] * f;
            x += *(const cf32x4_t *)&part[w][r][d] * f;
        }
        const int t = it.q0 + (it.row0 + r) / p.group, h = it.head * p.group + (it.row0 + r) % p.group;
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;   // nothing seen: 0
        struct alignas(4 * sizeof(T)) { T v[4]; } y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = (T)(x[e] * inverse);
        *(decltype(y) *)((T *)p.o + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + d) = y;
        if (d == 0) {
            const int64_t at = (int64_t)t * p.kv_heads * p.group + h;
            p.m[at] = mx * kLn2;
            p.l[at] = sum;
        }
    }
}

}  // namespace pmkl_amd
