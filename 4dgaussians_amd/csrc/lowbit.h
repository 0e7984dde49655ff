// Rows of numbers in 8 bits with one float32 scale per group of columns: the definition, shared by the row cache and the
// linear operator (lowbit.hip) and by the plane features that read the cache (hexplane.hip).
//
//   a = max |x| of the group     s = a / Q     inv = Q / a     code = round_fmt(x * inv)     value = s * code
//
// Q: the format's largest number.  The two quotients are IEEE divisions and the product and the rounding (half to even) are
// separate float32 operations, so the codes do not depend on the launch shape or on contraction.  s below 2^-126 (its
// reciprocal would overflow): the group is stored as zero.  An infinity or a NaN in a group makes s a NaN: the group reads
// as NaN instead of as numbers that were never written.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include "gs4d_internal.h"

typedef float lb_float2 __attribute__((ext_vector_type(2)));

template <int FMT> __device__ __forceinline__ constexpr float lb_top()
{
    return FMT == GS4D_FMT_INT8 ? 127.f : FMT == GS4D_FMT_E4M3 ? 448.f : FMT == GS4D_FMT_E5M2 ? 57344.f : 255.f;
}

struct LbScale { float s, inv; };

// amax_bits: max over the group of the values' bits without the sign, as unsigned numbers (a NaN is above infinity)
template <int FMT> __device__ __forceinline__ LbScale lb_scale(unsigned amax_bits)
{
    const float a = __uint_as_float(amax_bits), top = lb_top<FMT>();
    LbScale r;
    r.s = a / top;
    r.inv = top / a;
    if (r.s < 1.17549435e-38f) { r.s = 0.f; r.inv = 0.f; }
    if (amax_bits >= 0x7f800000u) { r.s = __uint_as_float(0x7fc00000u); r.inv = 0.f; }
    return r;
}

__device__ __forceinline__ unsigned lb_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// four quotients -> four codes in a word
template <int FMT> __device__ __forceinline__ unsigned lb_encode4(float a, float b, float c, float d)
{
    if constexpr (FMT == GS4D_FMT_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else if constexpr (FMT == GS4D_FMT_E5M2) {
        int w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    } else {
        const unsigned ia = (unsigned)(int)rintf(a), ib = (unsigned)(int)rintf(b), ic = (unsigned)(int)rintf(c), id = (unsigned)(int)rintf(d);
        return (ia & 255u) | (ib & 255u) << 8 | (ic & 255u) << 16 | id << 24;
    }
}

// the four codes of a word as float32 (exact)
template <int FMT> __device__ __forceinline__ float4 lb_decode4(unsigned w)
{
    if constexpr (FMT == GS4D_FMT_E4M3) {
        const lb_float2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return make_float4(lo[0], lo[1], hi[0], hi[1]);
    } else if constexpr (FMT == GS4D_FMT_E5M2) {
        const lb_float2 lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
        return make_float4(lo[0], lo[1], hi[0], hi[1]);
    } else if constexpr (FMT == GS4D_FMT_INT8) {
        return make_float4((float)(int)(signed char)w, (float)(int)(signed char)(w >> 8), (float)(int)(signed char)(w >> 16), (float)((int)w >> 24));
    } else {
        return make_float4((float)(w & 255u), (float)((w >> 8) & 255u), (float)((w >> 16) & 255u), (float)(w >> 24));
    }
}

// element types of the callers' tensors
struct LbBf16 { unsigned short v; };
struct LbF16 { _Float16 v; };
__device__ __forceinline__ float lb_load(float x) { return x; }
__device__ __forceinline__ float lb_load(LbBf16 x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float lb_load(LbF16 x) { return (float)x.v; }
template <typename T> __device__ __forceinline__ T lb_store(float x);
template <> __device__ __forceinline__ float lb_store<float>(float x) { return x; }
template <> __device__ __forceinline__ LbF16 lb_store<LbF16>(float x)
{
    asm("" : "+v"(x));                                   // the float32 number itself is rounded: a product must not be folded into the
    LbF16 r;                                             // conversion (v_fma_mixlo_f16 would round it once instead of twice)
    r.v = (_Float16)x;
    return r;
}
template <> __device__ __forceinline__ LbBf16 lb_store<LbBf16>(float x)
{
    LbBf16 r;
    const __bf16 b = (__bf16)x;                          // round to nearest even; a NaN stays one
    __builtin_memcpy(&r.v, &b, 2);
    return r;
}

static inline int lb_groups(int width, int group) { return (width + group - 1) / group; }

// One matrix of float32 rows kept as 8-bit rows (groups of 64 columns) and back: lowbit.hip, for the deformation field's checkpoint.
// x [rows][ld] (16-byte aligned, ld and width multiples of 4) <-> codes [rows][groups * 64], scales [rows][groups] and, rectified
// (relu: the values kept are max(x, 0)), bits [rows][groups][2] (bit c of a group: x > 0).  Read back, a rectified number whose bit
// is set is positive, whatever its code.  hmask (read only): the bits again, as rows of hld words at word hword + 2 * group, bit
// 4 m + q of word h standing for column 8 m + 4 h + q.
struct Gs4dKeepJob { float* x; int ld, width, relu; unsigned char* codes; float* scales; unsigned* bits; unsigned* hmask; int hld, hword; };
#define GS4D_KEEP_JOBS 12
struct Gs4dKeepJobs { Gs4dKeepJob j[GS4D_KEEP_JOBS]; int n, group0[GS4D_KEEP_JOBS + 1]; };
int gs4d_launch_keep(const Gs4dKeepJobs& jobs, long long rows, bool write, hipStream_t s);
