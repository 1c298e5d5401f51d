// What the cache kernels share: the cache's description, wave reductions and
// scans, and e4m3 conversions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pmkl_amd {

// pmkl_kv_cache with its strides filled in, in bytes but for the scales' heads.
struct CacheParams {
    uint8_t *k;
    uint8_t *v;
    float *k_scale;
    float *v_scale;
    int64_t k_sh, v_sh;     // head
    int64_t ks_sh, vs_sh;   // (elements)
    uint32_t k_sp, v_sp;    // page, below 2^31
    uint32_t ks_sp, vs_sp;
    int32_t k_st, v_sd;     // token of k, column of v
    int32_t pages;
    int32_t log2_page;
};

template <int CTRL>
__device__ __forceinline__ float cache_dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// Over the four 16-lane rows of a wave, every lane receiving the result of its
// column.
template <typename Op>
__device__ __forceinline__ float across_rows(float x, Op op) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

__device__ __forceinline__ float wave_max(float x) {
    const auto op = [](float a, float b) { return fmaxf(a, b); };
    x = op(x, cache_dpp<0xb1>(x));    // quad_perm 1 0 3 2
    x = op(x, cache_dpp<0x4e>(x));    // quad_perm 2 3 0 1
    x = op(x, cache_dpp<0x141>(x));   // row_half_mirror
    x = op(x, cache_dpp<0x140>(x));   // row_mirror
    return across_rows(x, op);
}

// Inclusive sums over the wave's lanes: within rows of 16, then the rows' sums
// to the rows behind.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast 15, to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast 31, to rows 2 and 3
    return x;
}
__device__ __forceinline__ int64_t wave_scan(int64_t x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

}  // namespace pmkl_amd
