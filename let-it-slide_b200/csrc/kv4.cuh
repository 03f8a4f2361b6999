// The KV cache in 4 bits (rptc_kv_cache, bits = 4): where a position's codes and scales lie, and its quantiser.
#pragma once
#include "common.cuh"

namespace rptc {

constexpr int kKv4Codes = 64;          // bytes of codes of a position and kv head (128 values)
constexpr int kKv4Scales = 16;         // bytes of scales: four groups of 32 values, (scale, minimum) each

inline int check_kv_cache(const rptc_kv_cache &c) {
    if (!c.k || !c.v || (c.bits != 4 && c.bits != 16)) return RPTC_ERR_ARG;
    if (c.bits == 4 && (!c.k_scales || !c.v_scales)) return RPTC_ERR_ARG;
    if (c.rows <= 0 || c.max_pos <= 0 || c.kv_heads <= 0) return RPTC_ERR_SHAPE;
    if (c.rows > 65535 || c.max_pos > (1 << 24) || c.kv_heads > 4096) return RPTC_ERR_TOO_LARGE;
    for (const void *p : {c.k, c.v, c.k_scales, c.v_scales})
        if (reinterpret_cast<uintptr_t>(p) & 15) return RPTC_ERR_ALIGN;
    return RPTC_OK;
}

#ifdef __CUDACC__
// NaN if either is.
__device__ __forceinline__ float kv4_min(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float kv4_max(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// A group's scale, as it is stored, and its reciprocal.  The difference and its fifteenth are rounded to 32 bits each, the scale then to fp16: what is stored is what the
// codes are counted in.  NaN where the range is NaN or infinite (the remainder is): all of a group stands for NaN as soon as one of its values is not finite, and what reads
// the cache shows it as it would an fp16 cache's.
__device__ __forceinline__ __half2 kv4_scale(float lo, float hi, float &inv) {
    const float range = hi - lo, part = range * (1.f / 15.f);
    const __half scale = __float2half_rn(fmaf(fmaf(-part, 15.f, range), 1.f / 15.f, part));      // the rounded fifteenth, for every significand
    const float step = __half2float(scale);
    inv = step > 0.f ? __frcp_rn(step) : 0.f;                                                      // scale 0: codes 0
    return __halves2half2(scale, __float2half_rn(lo));
}
// A value's code, as 12582912 + code: a sum of theirs and their multiples by 16, 256 and 4096 has the codes in its low 16 bits.
// The code is that of fp32 arithmetic, rounded half to even: v - lo rounded to 32 bits (the difference of two fp16 numbers may need some 40), over the scale, rounded to 32 bits.
// The quotient by Markstein's correction: an estimate by the correctly rounded reciprocal, its exact remainder by a fused multiply-add, and the remainder's quotient added,
// which is the correctly rounded quotient.  A difference that the first rounding brings to half-way between two codes goes to the even one: a minimum of -15, a scale of 2
// and a value of -1.8e-7 give 8, where unrounded numbers give 7 (7.5 less 2^-23).  The quotient passes 15.5 only where the scale was rounded by more than a thirtieth: below 2^-20
// (fp16's steps there are 2^-24), kKv4Exact with room to spare.
constexpr float kKv4Exact = 1.9073486328125e-6f;                     // 2^-19
__device__ __forceinline__ uint32_t kv4_code(float v, float lo, float step, float inv, bool small = true) {
    const float d = v - lo, q0 = d * inv, q = fmaf(fmaf(-q0, step, d), inv, q0);
    return __float_as_uint((small ? fminf(q, 15.f) : q) + 12582912.f);      // 1.5 * 2^23: rounds to the nearest whole number, half to even
}
// Eight neighbouring values of a thread, whose group of 32 is that of four neighbouring lanes -> the thread's eight codes (nibbles, first value lowest) and the
// group's scale and minimum.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&v)[8], __half2 &scale_min) {
    float lo = kv4_min(kv4_min(kv4_min(v[0], v[1]), kv4_min(v[2], v[3])), kv4_min(kv4_min(v[4], v[5]), kv4_min(v[6], v[7])));
    float hi = kv4_max(kv4_max(kv4_max(v[0], v[1]), kv4_max(v[2], v[3])), kv4_max(kv4_max(v[4], v[5]), kv4_max(v[6], v[7])));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = kv4_min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = kv4_max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    float inv;
    scale_min = kv4_scale(lo, hi, inv);
    const float step = __half2float(__low2half(scale_min));
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) codes |= (kv4_code(v[i], lo, step, inv) & 15u) << (4 * i);
    return codes;
}
#endif

}  // namespace rptc
