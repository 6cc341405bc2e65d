// wave.h -- exchanges between the lanes of a wave, in registers.
#pragma once

#include <hip/hip_runtime.h>

namespace qraf_hip {

template <int CTRL>
__device__ __forceinline__ int gdpp(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, true);
}
enum : int { GDPP_XOR1 = 0xB1, GDPP_XOR2 = 0x4E, GDPP_ROR4 = 0x124, GDPP_ROR8 = 0x128, GDPP_HALF_MIRROR = 0x141 };
// op over all lanes / over lanes l and l ^ 32, in every lane
template <typename T, typename F>
__device__ __forceinline__ T over_halves(T x, F op) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return op(__builtin_bit_cast(T, (unsigned)r[0]), __builtin_bit_cast(T, (unsigned)r[1]));
}
// (16 neighbouring lanes; lanes l and l ^ 16)
template <typename T, typename F>
__device__ __forceinline__ T over_row(T x, F op) {
    auto in = [](T v) { return __builtin_bit_cast(int, v); };
    auto back = [](int v) { return __builtin_bit_cast(T, v); };
    x = op(x, back(gdpp<GDPP_XOR1>(in(x))));
    x = op(x, back(gdpp<GDPP_XOR2>(in(x))));
    x = op(x, back(gdpp<GDPP_ROR4>(in(x))));
    return op(x, back(gdpp<GDPP_ROR8>(in(x))));
}
// (2, 4, 8 neighbouring lanes)
template <typename F>
__device__ __forceinline__ float over_pair(float x, F op) {
    return op(x, __int_as_float(gdpp<GDPP_XOR1>(__float_as_int(x))));
}
template <typename F>
__device__ __forceinline__ float over_quad(float x, F op) {
    x = over_pair(x, op);
    return op(x, __int_as_float(gdpp<GDPP_XOR2>(__float_as_int(x))));
}
template <typename F>
__device__ __forceinline__ float over_8(float x, F op) {
    x = over_quad(x, op);
    return op(x, __int_as_float(gdpp<GDPP_HALF_MIRROR>(__float_as_int(x))));
}
template <typename T, typename F>
__device__ __forceinline__ T over_rows(T x, F op) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return op(__builtin_bit_cast(T, (unsigned)r[0]), __builtin_bit_cast(T, (unsigned)r[1]));
}
template <typename T, typename F>
__device__ __forceinline__ T over_wave(T x, F op) {
    return over_halves(over_rows(over_row(x, op), op), op);
}

// the sum of a 64-bit value over all lanes, the same in every lane
__device__ __forceinline__ double wave_sum64(double x) {
    auto halves = [](double v, int& lo, int& hi) {
        lo = (int)__double_as_longlong(v);
        hi = (int)(__double_as_longlong(v) >> 32);
    };
    auto whole = [](unsigned lo, unsigned hi) { return __longlong_as_double((long long)hi << 32 | lo); };
    int lo, hi;
    halves(x, lo, hi);
    x += whole(gdpp<GDPP_XOR1>(lo), gdpp<GDPP_XOR1>(hi));
    halves(x, lo, hi);
    x += whole(gdpp<GDPP_XOR2>(lo), gdpp<GDPP_XOR2>(hi));
    halves(x, lo, hi);
    x += whole(gdpp<GDPP_ROR4>(lo), gdpp<GDPP_ROR4>(hi));
    halves(x, lo, hi);
    x += whole(gdpp<GDPP_ROR8>(lo), gdpp<GDPP_ROR8>(hi));
    halves(x, lo, hi);
    auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    x = whole(l[0], h[0]) + whole(l[1], h[1]);
    halves(x, lo, hi);
    l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    x = whole(l[0], h[0]) + whole(l[1], h[1]);
    halves(x, lo, hi);  // (rows rotated by 4 and 8 add in another order)
    return whole(__builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(hi));
}

}  // namespace qraf_hip
