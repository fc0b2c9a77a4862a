// Reductions over the lanes of a wavefront without LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace cfh {

// ---- reductions over a 16-lane row in DPP (VALU latency only; every lane must be active) --------
// quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror, row_mirror: after the four steps all
// 16 lanes of the row hold the reduction of the row.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_min(float x) {
    x = fminf(x, dpp_move<0xB1>(x));
    x = fminf(x, dpp_move<0x4E>(x));
    x = fminf(x, dpp_move<0x141>(x));
    x = fminf(x, dpp_move<0x140>(x));
    return x;
}
__device__ __forceinline__ float half_row_sum(float x) {      // over 8 lanes
    x += dpp_move<0xB1>(x);
    x += dpp_move<0x4E>(x);
    x += dpp_move<0x141>(x);
    return x;
}
__device__ __forceinline__ float row_sum(float x) {
    x = half_row_sum(x);
    x += dpp_move<0x140>(x);
    return x;
}

// ---- reductions over the four rows of a wavefront (same column), gfx950 lane swaps ---------------
// v_permlane32_swap exchanges the upper half of one register with the lower half of another,
// v_permlane16_swap the odd rows of one with the even rows of another: applied to two copies of x
// they hand every lane the two values to combine.  VALU only, no LDS round trip.
__device__ __forceinline__ void swap32(float x, float& lo, float& hi) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lo = __uint_as_float(r[0]); hi = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap16(float x, float& even, float& odd) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    even = __uint_as_float(r[0]); odd = __uint_as_float(r[1]);
}
__device__ __forceinline__ float rows_sum(float x) {      // every lane: sum over lanes c, c+16, c+32, c+48
    float p, q;
    swap32(x, p, q); x = p + q;
    swap16(x, p, q); return p + q;
}
__device__ __forceinline__ float rows_min(float x) {
    float p, q;
    swap32(x, p, q); x = fminf(p, q);
    swap16(x, p, q); return fminf(p, q);
}
// ---- wave64 reductions: rows in DPP, then across the rows -----------------------------------------
__device__ __forceinline__ float wave_sum(float v) { return rows_sum(row_sum(v)); }
__device__ __forceinline__ float wave_min(float v) { return rows_min(row_min(v)); }

}  // namespace cfh
