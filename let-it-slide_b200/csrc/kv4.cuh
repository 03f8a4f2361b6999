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
// Eight neighbouring values of a thread, whose group of 32 is that of four neighbouring lanes -> the thread's eight codes (nibbles, first value lowest) and the
// group's scale and minimum.  The difference, its fifteenth and the quotient are rounded to 32 bits each, the scale then to fp16: what is stored is
// what the codes are counted in.  A quotient differs from a half-way point by 2^-17 of itself at least (fp16 numbers over an fp16 number), which 32 bits hold.
__device__ __forceinline__ uint32_t kv4_quantise(const float (&v)[8], __half2 &scale_min) {
    float lo = v[0], hi = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    const __half scale = __float2half_rn(__fdiv_rn(hi - lo, 15.f));
    scale_min = __halves2half2(scale, __float2half_rn(lo));
    const float step = __half2float(scale);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = step > 0.f ? fminf(rintf(__fdiv_rn(v[i] - lo, step)), 15.f) : 0.f;
        codes |= (uint32_t)c << (4 * i);
    }
    return codes;
}
#endif

}  // namespace rptc
