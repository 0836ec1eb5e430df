// Running sums over a wave's 64 lanes by DPP: shifts by 1, 2, 4 and 8 inside the rows of 16, then the rows' last lanes handed on (a step of __shfl_up goes through LDS: 130 clocks against 8).
#pragma once

#include "pi_device.h"

template <int CTRL, int ROWS> static __device__ __forceinline__ uint32_t pi_scan_from(uint32_t v) { return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS> static __device__ __forceinline__ unsigned long long pi_scan_from(unsigned long long v) {
    return (unsigned long long) pi_scan_from<CTRL, ROWS>((uint32_t) (v >> 32)) << 32 | pi_scan_from<CTRL, ROWS>((uint32_t) v);
}
// what the lanes up to this one add up to (all 64 lanes call)
template <class T> static __device__ __forceinline__ T pi_wave_scan(T v) {
    v += pi_scan_from<0x111, 0xF>(v);                        // row_shr:1
    v += pi_scan_from<0x112, 0xF>(v);
    v += pi_scan_from<0x114, 0xF>(v);
    v += pi_scan_from<0x118, 0xF>(v);
    v += pi_scan_from<0x142, 0xA>(v);                        // row_bcast:15 to rows 1 and 3
    v += pi_scan_from<0x143, 0xC>(v);                        // row_bcast:31 to rows 2 and 3
    return v;
}
