// ft_wave.hpp -- sums, scans and maxima over a wavefront's 64 lanes, by DPP:
// within a row of 16 lanes by row shifts, then across the rows by the
// broadcasts of lanes 15 and 31 (row_bcast). A step takes a few cycles, where a
// shuffle through LDS takes about a hundred. Every lane of the wave has to be
// active; the results are the same on every run.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ft {

// The value `CTRL` moves to this lane; 0 where it moves none (rows out of ROWS included).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int wave_move0(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double wave_move0(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = wave_move0<CTRL, ROWS>((int)b), hi = wave_move0<CTRL, ROWS>((int)(b >> 32));
    return __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
}

// Sum of lanes 0..lane.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += wave_move0<0x111>(v);       // row_shr 1, 2, 4, 8
    v += wave_move0<0x112>(v);
    v += wave_move0<0x114>(v);
    v += wave_move0<0x118>(v);
    v += wave_move0<0x142, 0xA>(v);  // lane 15 of the row before to rows 1 and 3
    v += wave_move0<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}

__device__ __forceinline__ int wave_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ double wave_lane(double v, int l) {  // l: the same in every lane
    const long long b = __double_as_longlong(v);
    const int lo = wave_lane((int)b, l), hi = wave_lane((int)(b >> 32), l);
    return __longlong_as_double(((long long)hi << 32) | (uint32_t)lo);
}

// Sum of all lanes, in every lane.
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    return wave_lane(wave_scan(v), 63);
}

// The lane below's value; `first` in lane 0.
__device__ __forceinline__ double wave_lane_before(double v, double first) {
    const int lane = threadIdx.x & 63, from = lane ? lane - 1 : 0;
    const long long b = __double_as_longlong(v);
    const int lo = __shfl((int)b, from), hi = __shfl((int)(b >> 32), from);
    return lane ? __longlong_as_double(((long long)hi << 32) | (uint32_t)lo) : first;
}

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float wave_move(float v) {  // v itself where nothing moves here
    const int b = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(b, b, CTRL, ROWS, 0xF, false));
}

// Largest of a row's 16 lanes, in each of them, of a value that is no NaN: a
// step is one instruction, where fmaxf on a moved value takes three (the move
// and a maximum with itself, for signalling NaNs). A DPP operand may be read
// two wait states after it is written, also by what follows the asm, which the
// compiler does not look into.
__device__ __forceinline__ float row_max16(float v) {
    asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n\ts_nop 1"
        : "+v"(v));
    return v;
}

// The same of whole numbers; EIGHT: of 8 lanes.
template <bool EIGHT>
__device__ __forceinline__ uint32_t row_max16(uint32_t v) {
    asm("s_nop 1\n\tv_max_u32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\ts_nop 1"
        : "+v"(v));
    if (!EIGHT) asm("s_nop 1\n\tv_max_u32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n\ts_nop 1" : "+v"(v));
    return v;
}

// Largest of all lanes, in every lane; NaN is skipped.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, wave_move<0x111>(v));
    v = fmaxf(v, wave_move<0x112>(v));
    v = fmaxf(v, wave_move<0x114>(v));
    v = fmaxf(v, wave_move<0x118>(v));
    v = fmaxf(v, wave_move<0x142, 0xA>(v));
    v = fmaxf(v, wave_move<0x143, 0xC>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Lanes below this one that are in `set`.
__device__ __forceinline__ int wave_below(uint64_t set) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0));
}

// The value in scalar registers, whatever the compiler knows of it (as a
// literal, a constant of f64 costs two moves where it is used).
__device__ __forceinline__ double scalar(double v) {
    asm("" : "+s"(v));
    return v;
}

}  // namespace ft
