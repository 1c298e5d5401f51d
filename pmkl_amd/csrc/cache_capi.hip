// C ABI of the gfx950 key / value cache (include/pmkl_cache.h): argument
// checks, kernel choice and launches of the table builder, the append and the
// attention over the cache.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "cache_attn.hpp"
#include "cache_kernels.hpp"
#include "capi_common.hpp"
#include "pmkl_cache.h"

namespace {

using pmkl_amd::AppendParams;
using pmkl_amd::CacheAttnParams;
using pmkl_amd::CacheParams;
using pmkl_amd::SlotsParams;
using pmkl_capi::dtype_size;
using pmkl_capi::dtype_valid;

int check_page_size(int64_t ps) {
    PMKL_REQUIRE(ps >= PMKL_CACHE_MIN_PAGE_SIZE && ps <= PMKL_CACHE_MAX_PAGE_SIZE && (ps & (ps - 1)) == 0, PMKL_EINVAL,
                 "page_size %lld is not a power of two from %d to %d", (long long)ps, PMKL_CACHE_MIN_PAGE_SIZE,
                 PMKL_CACHE_MAX_PAGE_SIZE);
    return PMKL_OK;
}

int log2_of(int64_t v) {
    int r = 0;
    while ((int64_t(1) << r) < v) ++r;
    return r;
}

struct Dim {
    int64_t stride, size;
};

// Strides of a tensor: none negative, multiples of `vec`, and no offset past
// 2^62.  `written`: distinct positions must also not share an element; with the
// dimensions of size > 1 sorted by stride, each stride is at least the extent of
// those inside it.
int check_strides(const char *name, std::initializer_list<Dim> dims, int64_t inner, int64_t vec, bool written) {
    Dim sorted[4];
    int n = 0;
    double span = (double)inner;
    for (const Dim &d : dims) {
        PMKL_REQUIRE(d.stride >= 0 && d.stride % vec == 0, PMKL_EINVAL,
                     "%s stride %lld must be a non-negative multiple of %lld", name, (long long)d.stride, (long long)vec);
        span += (double)d.stride * (double)(d.size > 0 ? d.size - 1 : 0);
        if (d.size > 1) sorted[n++] = d;
    }
    PMKL_REQUIRE(span < 4.6e18, PMKL_EINVAL, "%s strides span too many elements", name);
    if (!written) return PMKL_OK;
    std::sort(sorted, sorted + n, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    int64_t extent = inner;
    for (int i = 0; i < n; ++i) {
        PMKL_REQUIRE(sorted[i].stride >= extent, PMKL_EINVAL, "%s strides make distinct rows overlap", name);
        extent += sorted[i].stride * (sorted[i].size - 1);
    }
    return PMKL_OK;
}

int check_pointer(const char *name, const void *p, size_t align) {
    PMKL_REQUIRE(p != nullptr, PMKL_EINVAL, "%s is a null pointer", name);
    PMKL_REQUIRE((uintptr_t)p % align == 0, PMKL_EINVAL, "%s must be %d-byte aligned", name, (int)align);
    return PMKL_OK;
}

#define PMKL_TRY(expr)                       \
    do {                                     \
        const int rc_ = (expr);              \
        if (rc_ != PMKL_OK) return rc_;      \
    } while (0)

bool all_zero(const int64_t *s, int n) {
    return std::all_of(s, s + n, [](int64_t x) { return x == 0; });
}

// The shape alone: what decides support and launch shapes.
int check_cache_shape(const pmkl_kv_cache &c) {
    PMKL_TRY(check_page_size(c.page_size));
    PMKL_REQUIRE(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128, PMKL_EUNSUPPORTED,
                 "head_dim %lld has no compiled kernel (supported: 32, 64, 128)", (long long)c.head_dim);
    PMKL_REQUIRE(c.kv_heads >= 1 && c.kv_heads <= 65535, PMKL_EINVAL, "kv_heads %lld is not in 1 .. 65535",
                 (long long)c.kv_heads);
    PMKL_REQUIRE(c.pages >= 0 && c.pages <= INT32_MAX, PMKL_EINVAL, "pages %lld is not in 0 .. 2^31 - 1",
                 (long long)c.pages);
    return PMKL_OK;
}

// Strides and pointers of a cache with work to do.  written: the call stores
// into it.
int fill_cache(const pmkl_kv_cache &c, bool written, CacheParams *p) {
    PMKL_REQUIRE(c.pages > 0, PMKL_EINVAL, "a cache of no pages");
    const int64_t P = c.pages, H = c.kv_heads, ps = c.page_size, D = c.head_dim;
    int64_t ks[3], vs[3], kss[2], vss[2];
    memcpy(ks, c.k_strides, sizeof(ks));
    memcpy(vs, c.v_strides, sizeof(vs));
    memcpy(kss, c.k_scale_strides, sizeof(kss));
    memcpy(vss, c.v_scale_strides, sizeof(vss));
    if (all_zero(ks, 3)) ks[0] = H * ps * D, ks[1] = ps * D, ks[2] = D;
    if (all_zero(vs, 3)) vs[0] = H * ps * D, vs[1] = ps * D, vs[2] = ps;
    if (all_zero(kss, 2)) kss[0] = H, kss[1] = 1;
    if (all_zero(vss, 2)) vss[0] = H, vss[1] = 1;
    PMKL_TRY(check_pointer("k_cache", c.k, 16));
    PMKL_TRY(check_pointer("v_cache", c.v, 16));
    PMKL_TRY(check_pointer("k_scale", c.k_scale, 4));
    PMKL_TRY(check_pointer("v_scale", c.v_scale, 4));
    // inside a page the kernels' offsets are 32 bits
    PMKL_REQUIRE(ks[2] <= INT32_MAX / ps && vs[2] <= INT32_MAX / D, PMKL_EINVAL,
                 "a page's tokens or columns span more than 2 GiB");
    PMKL_TRY(check_strides("k_cache", {{ks[0], P}, {ks[1], H}, {ks[2], ps}}, D, 16, written));
    PMKL_TRY(check_strides("v_cache", {{vs[0], P}, {vs[1], H}, {vs[2], D}}, ps, 16, written));
    PMKL_TRY(check_strides("k_scale", {{kss[0], P}, {kss[1], H}}, 1, 1, written));
    PMKL_TRY(check_strides("v_scale", {{vss[0], P}, {vss[1], H}}, 1, 1, written));
    PMKL_REQUIRE(ks[0] <= INT32_MAX && vs[0] <= INT32_MAX && kss[0] <= INT32_MAX / 4 && vss[0] <= INT32_MAX / 4,
                 PMKL_EINVAL, "pages lie more than 2 GiB apart");
    p->k = (uint8_t *)c.k;
    p->v = (uint8_t *)c.v;
    p->k_scale = c.k_scale;
    p->v_scale = c.v_scale;
    p->k_sp = (uint32_t)ks[0], p->k_sh = ks[1], p->k_st = (int32_t)ks[2];
    p->v_sp = (uint32_t)vs[0], p->v_sh = vs[1], p->v_sd = (int32_t)vs[2];
    p->ks_sp = (uint32_t)(kss[0] * 4), p->ks_sh = kss[1];
    p->vs_sp = (uint32_t)(vss[0] * 4), p->vs_sh = vss[1];
    p->pages = (int32_t)P;
    p->log2_page = log2_of(ps);
    return PMKL_OK;
}

int launched(const char *what) {
    const hipError_t err = hipGetLastError();
    PMKL_REQUIRE(err == hipSuccess, PMKL_EHIP, "%s launch failed: %s", what, hipGetErrorString(err));
    return PMKL_OK;
}

struct Range {
    const char *name;
    const void *p;
    uint64_t bytes;
};

int check_disjoint(const Range &out, const Range &in) {
    const uintptr_t a = (uintptr_t)out.p, b = (uintptr_t)in.p;
    PMKL_REQUIRE(a + out.bytes <= b || b + in.bytes <= a, PMKL_EINVAL, "%s overlaps %s", out.name, in.name);
    return PMKL_OK;
}

int run_slots(const pmkl_cache_slots_args *a, void *stream) {
    PMKL_REQUIRE(a != nullptr, PMKL_EINVAL, "args is a null pointer");
    PMKL_TRY(check_page_size(a->page_size));
    PMKL_REQUIRE(a->batch >= 0 && a->batch <= INT32_MAX && a->table_width >= 0 && a->table_width <= INT32_MAX &&
                     a->free_count >= 0 && a->free_count <= INT32_MAX && a->tokens >= 0 && a->tokens <= INT32_MAX,
                 PMKL_EINVAL, "batch %lld, table_width %lld, free_count %lld and tokens %lld must be in 0 .. 2^31 - 1",
                 (long long)a->batch, (long long)a->table_width, (long long)a->free_count, (long long)a->tokens);
    const int64_t stride = a->table_stride ? a->table_stride : a->table_width;
    PMKL_REQUIRE(a->batch <= 1 || stride >= a->table_width, PMKL_EINVAL, "table_stride %lld < table_width %lld",
                 (long long)stride, (long long)a->table_width);
    PMKL_REQUIRE(stride >= 0 && stride <= (int64_t(1) << 40), PMKL_EINVAL, "table_stride %lld is not in 0 .. 2^40",
                 (long long)stride);
    if (a->batch > 0) {
        PMKL_TRY(check_pointer("cached_lens", a->cached_lens, 4));
        PMKL_TRY(check_pointer("new_lens", a->new_lens, 4));
        PMKL_TRY(check_pointer("seq_lens", a->seq_lens, 4));
        if (a->table_width > 0) PMKL_TRY(check_pointer("block_table", a->block_table, 4));
    }
    if (a->free_count > 0) PMKL_TRY(check_pointer("free_pages", a->free_pages, 4));
    if (a->tokens > 0) PMKL_TRY(check_pointer("slots", a->slots, 8));
    PMKL_TRY(check_pointer("free_head", a->free_head, 4));
    PMKL_TRY(check_pointer("query_start", a->query_start, 4));
    PMKL_TRY(check_pointer("free_head_out", a->free_head_out, 4));
    // every workgroup reads all inputs while others write
    const uint64_t B = (uint64_t)a->batch * 4;
    const uint64_t table = a->batch ? ((uint64_t)(a->batch - 1) * stride + a->table_width) * 4 : 0;
    const Range outs[] = {{"seq_lens", a->seq_lens, B}, {"query_start", a->query_start, B + 4},
                          {"slots", a->slots, (uint64_t)a->tokens * 8}, {"free_head_out", a->free_head_out, 4},
                          {"block_table", a->block_table, table}};
    const Range ins[] = {{"cached_lens", a->cached_lens, B}, {"new_lens", a->new_lens, B},
                         {"free_pages", a->free_pages, (uint64_t)a->free_count * 4}, {"free_head", a->free_head, 4}};
    for (size_t i = 0; i < sizeof(outs) / sizeof(*outs); ++i) {
        for (const Range &in : ins)
            if (outs[i].bytes && in.bytes) PMKL_TRY(check_disjoint(outs[i], in));
        for (size_t j = 0; j < i; ++j)
            if (outs[i].bytes && outs[j].bytes) PMKL_TRY(check_disjoint(outs[i], outs[j]));
    }

    SlotsParams p;
    p.cached_lens = a->cached_lens;
    p.new_lens = a->new_lens;
    p.table = a->block_table;
    p.free_pages = a->free_pages;
    p.free_head = a->free_head;
    p.seq_lens = a->seq_lens;
    p.query_start = a->query_start;
    p.slots = a->slots;
    p.free_head_out = a->free_head_out;
    p.table_stride = stride;
    p.free_count = a->free_count;
    p.tokens = a->tokens;
    p.batch = (int32_t)a->batch;
    p.width = (int32_t)a->table_width;
    p.log2_page = log2_of(a->page_size);
    constexpr int NT = pmkl_amd::kCacheThreads;
    const int64_t blocks = std::max((a->tokens + NT - 1) / NT, (a->batch + NT - 1) / NT);
    const int64_t grid = std::min<int64_t>(std::max<int64_t>(blocks, 1), 512);
    hipLaunchKernelGGL(pmkl_amd::cache_slots_kernel, dim3((unsigned)grid), dim3(NT), 0, (hipStream_t)stream, p);
    return launched("cache_slots");
}

typedef void (*append_fn)(AppendParams);

template <typename T>
append_fn pick_append(int64_t D) {
    switch (D) {
        case 32: return pmkl_amd::cache_append_kernel<T, 32>;
        case 64: return pmkl_amd::cache_append_kernel<T, 64>;
        default: return pmkl_amd::cache_append_kernel<T, 128>;
    }
}

int run_append(const pmkl_cache_append_args *a, void *stream) {
    PMKL_REQUIRE(a != nullptr, PMKL_EINVAL, "args is a null pointer");
    PMKL_REQUIRE(dtype_valid(a->dtype), PMKL_EUNSUPPORTED, "unsupported dtype %d", (int)a->dtype);
    PMKL_TRY(check_cache_shape(a->cache));
    PMKL_REQUIRE(a->tokens >= 0 && a->tokens <= INT32_MAX, PMKL_EINVAL, "tokens %lld is not in 0 .. 2^31 - 1",
                 (long long)a->tokens);
    if (a->tokens == 0) return PMKL_OK;
    AppendParams p;
    PMKL_TRY(fill_cache(a->cache, true, &p.cache));
    const int64_t H = a->cache.kv_heads, D = a->cache.head_dim, vec = 16 / (int64_t)dtype_size(a->dtype);
    PMKL_TRY(check_pointer("k", a->k, 16));
    PMKL_TRY(check_pointer("v", a->v, 16));
    PMKL_TRY(check_pointer("slots", a->slots, 8));
    const bool ck = all_zero(a->k_strides, 2), cv = all_zero(a->v_strides, 2);
    p.k = a->k;
    p.v = a->v;
    p.slots = a->slots;
    p.k_st = ck ? H * D : a->k_strides[0], p.k_sh = ck ? D : a->k_strides[1];
    p.v_st = cv ? H * D : a->v_strides[0], p.v_sh = cv ? D : a->v_strides[1];
    PMKL_TRY(check_strides("k", {{p.k_st, a->tokens}, {p.k_sh, H}}, D, vec, false));
    PMKL_TRY(check_strides("v", {{p.v_st, a->tokens}, {p.v_sh, H}}, D, vec, false));
    p.tokens = a->tokens;
    p.kv_heads = (int32_t)H;
    // Of 64 tokens between 64 runs (decoding) and 1 (a prompt in large pages)
    // begin; each is 2 H wave items.  About 8,192 waves in all keep the card
    // busy; more, where a window of a prompt needs them for a page each, and no
    // more than the items of 64 runs.  In large pages four waves may share an item.
    const int64_t windows = (a->tokens + 63) / 64, waves = pmkl_amd::kCacheThreads / 64;
    const int64_t runs = std::min<int64_t>(64, a->tokens), pages = std::min<int64_t>(runs, 64 / a->cache.page_size + 1);
    const int64_t per = a->cache.page_size >= 64 ? 1 : waves;   // items of a workgroup
    const int64_t y = std::max<int64_t>({1, std::min(runs * 2 * H / per, 8192 / waves / windows), pages * 2 * H / per});
    const append_fn fn = a->dtype == PMKL_DTYPE_F32 ? pick_append<float>(D)
                         : a->dtype == PMKL_DTYPE_F16 ? pick_append<_Float16>(D) : pick_append<__bf16>(D);
    PMKL_REQUIRE(windows * y * pmkl_amd::kCacheThreads < (int64_t(1) << 32), PMKL_EINVAL, "grid too large");
    hipLaunchKernelGGL(fn, dim3((unsigned)windows, (unsigned)y), dim3(pmkl_amd::kCacheThreads), 0, (hipStream_t)stream, p);
    return launched("cache_append");
}

typedef void (*cache_attn_fn)(CacheAttnParams);
constexpr int kAttnWaves = 4;
constexpr int64_t kChunkRows = pmkl_amd::kChunkRows;

// The join's waves of a workgroup and ranges that it looks at.
struct JoinShape {
    int waves, per;
};
constexpr JoinShape kJoins[3] = {{4, 1}, {8, 2}, {16, 4}};

struct AttnKernels {
    cache_attn_fn whole, split, chunk, joins[3];
    int split_waves;   // that a SIMD holds of `split`
};

template <typename T, int D>
AttnKernels attn_kernels() {
    return {pmkl_amd::cache_attn_kernel<T, D, kAttnWaves>, pmkl_amd::cache_attn_split_kernel<T, D>,
            pmkl_amd::cache_attn_chunk_kernel<T, D>,
            {pmkl_amd::cache_attn_join_kernel<T, D, kJoins[0].waves, kJoins[0].per>,
             pmkl_amd::cache_attn_join_kernel<T, D, kJoins[1].waves, kJoins[1].per>,
             pmkl_amd::cache_attn_join_kernel<T, D, kJoins[2].waves, kJoins[2].per>},
            pmkl_amd::cache_split_waves<T, D>()};
}
template <typename T>
AttnKernels pick_attn(int64_t D) {
    switch (D) {
        case 32: return attn_kernels<T, 32>();
        case 64: return attn_kernels<T, 64>();
        default: return attn_kernels<T, 128>();
    }
}

struct AttnPlan {
    AttnKernels fn;
    bool split;
    int64_t grid, threads, ranges;
    int join;         // which of kJoins
    int64_t chunks;   // workgroups of the chunks' form, beside the split one; 0: it is not used
    uint64_t parts, workspace;   // bytes: of the split form's parts, in all
    bool empty;
};

// The shape of a call: which kernels and how many workgroups.  Looks at no
// pointer.
int plan_attn(const pmkl_cache_attn_args *a, AttnPlan *pl) {
    *pl = AttnPlan{};
    PMKL_REQUIRE(a != nullptr, PMKL_EINVAL, "args is a null pointer");
    PMKL_REQUIRE(dtype_valid(a->dtype), PMKL_EUNSUPPORTED, "unsupported dtype %d", (int)a->dtype);
    PMKL_TRY(check_cache_shape(a->cache));
    PMKL_REQUIRE(std::isfinite(a->scale) && a->scale >= 0.f, PMKL_EINVAL, "scale must be finite and >= 0");
    PMKL_REQUIRE(a->batch >= 0 && a->batch <= INT32_MAX && a->table_width >= 0 && a->table_width <= INT32_MAX &&
                     a->tokens >= 0 && a->heads >= 0,
                 PMKL_EINVAL, "batch %lld and table_width %lld must be in 0 .. 2^31 - 1, tokens %lld and heads %lld not "
                 "negative", (long long)a->batch, (long long)a->table_width, (long long)a->tokens, (long long)a->heads);
    PMKL_REQUIRE(a->table_width * a->cache.page_size <= INT32_MAX - 256, PMKL_EINVAL,
                 "table_width %lld * page_size %lld is past 2^31 tokens", (long long)a->table_width,
                 (long long)a->cache.page_size);
    PMKL_REQUIRE(a->heads % a->cache.kv_heads == 0, PMKL_EINVAL, "heads %lld is not a multiple of kv_heads %lld",
                 (long long)a->heads, (long long)a->cache.kv_heads);
    PMKL_REQUIRE(a->heads <= INT32_MAX && a->tokens <= INT32_MAX / std::max<int64_t>(a->heads, 1), PMKL_EINVAL,
                 "tokens %lld * heads %lld is past 2^31 - 1", (long long)a->tokens, (long long)a->heads);
    if (a->batch == 0 || a->tokens == 0 || a->heads == 0) {
        pl->empty = true;
        return PMKL_OK;
    }
    const int64_t D = a->cache.head_dim, G = a->heads / a->cache.kv_heads;
    pl->fn = a->dtype == PMKL_DTYPE_F32 ? pick_attn<float>(D)
             : a->dtype == PMKL_DTYPE_F16 ? pick_attn<_Float16>(D) : pick_attn<__bf16>(D);
    // every request's last block may be partly filled; a request without tokens has none
    pl->grid = (a->tokens * G / pmkl_amd::kCacheRows + std::min(a->batch, a->tokens)) * a->cache.kv_heads;
    // the split form counts tiles of all row blocks in 32 bits
    const int64_t tiles = (a->table_width * a->cache.page_size + pmkl_amd::kCacheTile - 1) / pmkl_amd::kCacheTile +
                          pmkl_amd::kBlockCost;
    pl->threads = kAttnWaves * 64;
    // Chunks have their own form where rows are enough for a workgroup of 128 on every
    // CU, and by as much more as a row costs less: a workgroup's tiles take their time
    // however few there are.  us, and in the split form alone: head_dim 128 in bf16,
    // 16,384 rows of all heads 69, 49; 24,576: 68, 68; 32,768: 69, 84; 65,536: 74, 122; in
    // fp32 32,768: 99, 132; head_dim 64 at 65,536 71, 73 (fp32 103, 128); head_dim 32 at
    // 131,072 73, 78.  A call of single tokens has none.
    const int64_t heads = a->cache.kv_heads, rows = a->tokens * G;
    const bool many = a->tokens >= 2 * a->batch;
    if (many && rows * heads * D >= kChunkRows * 256 * 128)
        pl->chunks = (rows / kChunkRows + std::min(std::min(a->batch, a->tokens), rows / kChunkRows)) * heads;
    // A table for so few tokens is not worth a second launch, to join: a request of 1,024
    // keys 13.2 us and 12.5 split, 512 keys 8.6 and 11.7, 2,048 keys 21.6 and 13.3
    // (head_dim 128); 1,536 keys of head_dim 64 12.6 and 12.1, 1,024 keys 9.0 and 13.8.
    pl->split = (a->table_width * a->cache.page_size > (D >= 128 ? 1024 : 1536) || pl->chunks) && pl->grid <= INT32_MAX / tiles;
    if (!pl->split) pl->chunks = 0;
    if (pl->split) {
        const int64_t blocks = pl->grid;
        // As many waves as the chip's 1,024 SIMDs hold of the kernel.  But single tokens of
        // head_dim 128 are bound by loads, and one wave a SIMD has as many on the way as
        // the memory takes (bf16, 16 requests of 4 k 20.1 us, with two 21.6; 128 of 16 k
        // 177.6 and 176.8) and leaves half as many parts (4 of 4 k: 18.1 and 20.9); rows of
        // a chunk are bound by arithmetic (256 tokens: 122 and 102).
        pl->ranges = 1024 * (D >= 128 && !many ? 1 : pl->fn.split_waves);
        pl->grid = pl->ranges / pmkl_amd::kSplitWaves;
        pl->threads = pmkl_amd::kSplitWaves * 64;
        pl->parts = (uint64_t)2 * pl->ranges * pmkl_amd::kCacheRows * (D + 2) * sizeof(float);
        pl->workspace = pl->parts + pl->ranges * sizeof(pmkl_amd::CacheUnfinished);
        // at most so many blocks have parts, and all of them together few more parts than ranges
        pl->join = blocks * 64 < pl->ranges ? 2 : blocks * 8 < pl->ranges ? 1 : 0;
    }
    PMKL_REQUIRE(pl->grid * pl->threads < (int64_t(1) << 32) && pl->chunks * pmkl_amd::kChunkWaves * 64 < (int64_t(1) << 32),
                 PMKL_EINVAL, "grid too large (%lld workgroups)", (long long)std::max(pl->grid, pl->chunks));
    return PMKL_OK;
}

int run_attn(const pmkl_cache_attn_args *a, void *stream) {
    AttnPlan pl;
    PMKL_TRY(plan_attn(a, &pl));
    if (pl.empty) return PMKL_OK;
    const int64_t H = a->heads, D = a->cache.head_dim, vec = 16 / (int64_t)dtype_size(a->dtype);
    CacheAttnParams p;
    PMKL_TRY(fill_cache(a->cache, false, &p.cache));
    PMKL_TRY(check_pointer("q", a->q, 16));
    PMKL_TRY(check_pointer("o", a->o, 16));
    PMKL_TRY(check_pointer("m", a->m, 4));
    PMKL_TRY(check_pointer("l", a->l, 4));
    PMKL_TRY(check_pointer("seq_lens", a->seq_lens, 4));
    PMKL_TRY(check_pointer("query_start", a->query_start, 4));
    if (a->table_width > 0) PMKL_TRY(check_pointer("block_table", a->block_table, 4));
    const bool cq = all_zero(a->q_strides, 2), co = all_zero(a->o_strides, 2);
    p.q_st = cq ? H * D : a->q_strides[0], p.q_sh = cq ? D : a->q_strides[1];
    p.o_st = co ? H * D : a->o_strides[0], p.o_sh = co ? D : a->o_strides[1];
    PMKL_TRY(check_strides("q", {{p.q_st, a->tokens}, {p.q_sh, H}}, D, vec, false));
    PMKL_TRY(check_strides("o", {{p.o_st, a->tokens}, {p.o_sh, H}}, D, vec, true));
    p.table_stride = a->table_stride ? a->table_stride : a->table_width;
    PMKL_REQUIRE(p.table_stride >= 0 && p.table_stride <= (int64_t(1) << 40), PMKL_EINVAL,
                 "table_stride %lld is not in 0 .. 2^40", (long long)p.table_stride);
    if (pl.split) {
        PMKL_TRY(check_pointer("workspace", a->workspace, 16));
        PMKL_REQUIRE(a->workspace_bytes >= pl.workspace, PMKL_EINVAL, "workspace of %llu bytes is too small (needs %llu)",
                     (unsigned long long)a->workspace_bytes, (unsigned long long)pl.workspace);
    }
    p.parts = (float *)a->workspace;
    p.unfinished = (pmkl_amd::CacheUnfinished *)((char *)a->workspace + pl.parts);
    p.q = a->q;
    p.o = a->o;
    p.m = a->m;
    p.l = a->l;
    p.table = a->block_table;
    p.seq_lens = a->seq_lens;
    p.query_start = a->query_start;
    p.tokens = (int32_t)a->tokens;
    p.batch = (int32_t)a->batch;
    p.width = (int32_t)a->table_width;
    p.kv_heads = (int32_t)a->cache.kv_heads;
    p.group = (int32_t)(H / a->cache.kv_heads);
    p.is_causal = a->is_causal ? 1 : 0;
    p.scale = a->scale > 0.f ? a->scale : 1.0f / std::sqrt((float)D);
    p.ranges = (int32_t)pl.ranges;
    p.chunks = pl.chunks ? 1 : 0;
    hipLaunchKernelGGL(pl.split ? pl.fn.split : pl.fn.whole, dim3((unsigned)pl.grid), dim3((unsigned)pl.threads), 0,
                       (hipStream_t)stream, p);
    PMKL_TRY(launched("cache_attn"));
    if (!pl.split) return PMKL_OK;
    if (pl.chunks) {
        hipLaunchKernelGGL(pl.fn.chunk, dim3((unsigned)pl.chunks), dim3(pmkl_amd::kChunkWaves * 64), 0, (hipStream_t)stream, p);
        PMKL_TRY(launched("cache_attn_chunk"));
    }
    const JoinShape join = kJoins[pl.join];
    hipLaunchKernelGGL(pl.fn.joins[pl.join], dim3((unsigned)(pl.ranges / join.per)), dim3((unsigned)join.waves * 64), 0,
                       (hipStream_t)stream, p);
    return launched("cache_attn_join");
}

}  // namespace

extern "C" {

int pmkl_cache_slots(const pmkl_cache_slots_args *a, void *stream) {
    pmkl_capi::g_err[0] = '\0';
    return run_slots(a, stream);
}

int pmkl_cache_append(const pmkl_cache_append_args *a, void *stream) {
    pmkl_capi::g_err[0] = '\0';
    return run_append(a, stream);
}

int pmkl_cache_attn_fwd(const pmkl_cache_attn_args *a, void *stream) {
    pmkl_capi::g_err[0] = '\0';
    return run_attn(a, stream);
}

uint64_t pmkl_cache_attn_workspace_size(const pmkl_cache_attn_args *a) {
    pmkl_capi::g_err[0] = '\0';
    AttnPlan pl;
    return plan_attn(a, &pl) == PMKL_OK ? pl.workspace : 0;
}

const char *pmkl_cache_attn_kernel_name(const pmkl_cache_attn_args *a) {
    pmkl_capi::g_err[0] = '\0';
    static thread_local char name[200];
    AttnPlan pl;
    if (plan_attn(a, &pl) != PMKL_OK) return nullptr;
    if (pl.empty) return "none";
    const char *dt = a->dtype == PMKL_DTYPE_BF16 ? "bf16" : a->dtype == PMKL_DTYPE_F16 ? "fp16" : "fp32";
    const long long D = a->cache.head_dim;
    int n = snprintf(name, sizeof(name), "cache_attn_%skernel<%s, %lld> grid %lld x %d", pl.split ? "split_" : "", dt, D,
                     (long long)pl.grid, (int)pl.threads);
    if (pl.chunks)
        n += snprintf(name + n, sizeof(name) - n, ", cache_attn_chunk_kernel<%s, %lld> grid %lld x %d", dt, D,
                      (long long)pl.chunks, pmkl_amd::kChunkWaves * 64);
    if (pl.split)
        snprintf(name + n, sizeof(name) - n, ", cache_attn_join_kernel<%s, %lld, %d, %d> grid %lld x %d", dt, D, kJoins[pl.join].waves,
                 kJoins[pl.join].per, (long long)(pl.ranges / kJoins[pl.join].per), kJoins[pl.join].waves * 64);
    return name;
}

}  // extern "C"
