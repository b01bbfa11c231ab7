// What the sequence operators share (recurrence.hip, rows.hip, scores.hip): the storage types of include/dcarl.h (DCARL_F64 ... DCARL_F16), the
// type their sums are held in (f32; f64 for f64 storage), element conversions.  These units are compiled with NaNs honoured
// (build.py SOURCE_FLAGS): a NaN is an ordinary input here.
#pragma once
#include "common.h"

namespace dcarl {

struct bf16 { uint16_t bits; };
struct f16 { _Float16 v; };

template <typename T> struct SeqType;                       // Acc: what sums, states and products are held in
template <> struct SeqType<double> { using Acc = double; };
template <> struct SeqType<float> { using Acc = float; };
template <> struct SeqType<bf16> { using Acc = float; };
template <> struct SeqType<f16> { using Acc = float; };

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float widen(f16 v) { return (float)v.v; }
// the one rounding of a result: to nearest, ties to even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T, typename A> __device__ __forceinline__ T narrow(A v) {
    if constexpr (__is_same(T, bf16)) return bf16{__builtin_bit_cast(uint16_t, (__bf16)(float)v)};
    else if constexpr (__is_same(T, f16)) return f16{(_Float16)(float)v};
    else return (T)v;
}

// calls f(T{}) for the storage type `type`; the entry points have checked that it is one of the four
template <typename F> inline void with_type(int type, F&& f) {
    switch (type) {
        case DCARL_F64: f(double{}); break;
        case DCARL_F32: f(float{}); break;
        case DCARL_BF16: f(bf16{}); break;
        default: f(f16{}); break;
    }
}

}  // namespace dcarl
