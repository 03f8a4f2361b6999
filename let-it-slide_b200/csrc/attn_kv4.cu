// Single-query attention over a KV cache in 4 bits (rptc_kv_cache, bits = 4).  No reference counterpart.
#include "fwht.cuh"
#include "kv4.cuh"

namespace rptc {

struct AttnKv4Params {
    const __half *q;
    int64_t ld_q;
    const int32_t *pos;
    const uint8_t *k, *v;
    const __half2 *k_scales, *v_scales;
    __half *out;
    int64_t ld_out, max_pos;
    int32_t hq, hkv;
    float scale;
    const __half *signs_in;
    unsigned int *status;
};

// One CTA of four warps per (row, q head); eight lanes take a position, a lane four dims of each group.
__global__ void __launch_bounds__(128) attn_kv4_kernel(const AttnKv4Params p) {
    __shared__ float part[16][128], pm[16], pl[16], tr[128];
    pdl_allow_next_grid();
    pdl_wait_prior_grids();
    const int row = blockIdx.y, head = blockIdx.x, kvh = head / (p.hq / p.hkv), t = threadIdx.x, g = t & 7, grp = t >> 3;
    const int pos = __ldg(after_wait(p.pos) + row);
    __half *out = p.out + (int64_t)row * p.ld_out + head * 128;
    if (pos < 0 || pos >= p.max_pos) {
        if (pos != -1 && t == 0) atomicExch(p.status, kStatusPosition);
        out[t] = __float2half_rn(0.f);
        return;
    }
    float q[16], acc[16] = {}, m = -INFINITY, l = 0.f;
    const __half *qp = after_wait(p.q) + (int64_t)row * p.ld_q + head * 128;
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = __half2float(qp[32 * (i >> 2) + 4 * g + (i & 3)]) * p.scale * 1.4426950408889634f;
    for (int j0 = 0; j0 <= pos; j0 += 16) {
        const int j = j0 + grp;
        const int64_t at = ((int64_t)row * p.hkv + kvh) * p.max_pos + min(j, pos);
        auto values = [&](const uint8_t *c, const __half2 *s, float (&x)[16]) {
            const uint2 w = *reinterpret_cast<const uint2 *>(c + at * kKv4Codes + 8 * g);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 f = __half22float2(s[at * 4 + (i >> 2)]);
                x[i] = fmaf((float)(((i < 8 ? w.x : w.y) >> (4 * (i & 7))) & 15u), f.x, f.y);
            }
        };
        float x[16], s = 0.f;
        values(after_wait(p.k), after_wait(p.k_scales), x);
#pragma unroll
        for (int i = 0; i < 16; ++i) s = fmaf(q[i], x[i], s);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (j > pos) continue;                               // of eight lanes, which meet again at the next shuffle
        const float mn = fmaxf(m, s), f = exp2f(m - mn), e = exp2f(s - mn);
        values(after_wait(p.v), after_wait(p.v_scales), x);
        l = l * f + e;
        m = mn;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = fmaf(e, x[i], acc[i] * f);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) part[grp][32 * (i >> 2) + 4 * g + (i & 3)] = acc[i];
    if (g == 0) pm[grp] = m, pl[grp] = l;
    __syncthreads();
    float mx = pm[0], num = 0.f, den = 0.f;
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, pm[i]);
    for (int i = 0; i < 16; ++i) {
        const float f = exp2f(pm[i] - mx);
        num += part[i][t] * f;
        den += pl[i] * f;
    }
    float o = num / den;
    if (p.signs_in) {
        tr[t] = __half2float(__float2half_rn(o)) * __half2float(p.signs_in[head * 128 + t]);
        __syncthreads();
        o = 0.f;
        for (int i = 0; i < 128; ++i) o += (__popc(i & t) & 1) ? -tr[i] : tr[i];
        o *= hadamard_norm_dev(128);
    }
    out[t] = __float2half_rn(o);
}

}  // namespace rptc

using namespace rptc;

extern "C" int64_t rptc_attn_decode_kv4_workspace_bytes(const rptc_kv_cache *cache, int heads) {
    (void)cache, (void)heads;
    return 0;
}

extern "C" int rptc_attn_decode_kv4(const void *q, int64_t ld_q, const int32_t *pos, const rptc_kv_cache *cache, void *out, int64_t ld_out, int heads,
                                    float scale, const void *signs_in, void *workspace, int64_t workspace_bytes, rptc_stream_t stream) {
    if (!q || !pos || !cache || !out) return RPTC_ERR_ARG;
    if (int e = check_kv_cache(*cache)) return e;
    if (cache->bits != 4) return RPTC_ERR_UNSUPPORTED;
    if (!(scale > 0.f && scale < 1e30f)) return RPTC_ERR_ARG;
    if (heads <= 0 || heads % cache->kv_heads || ld_q < (int64_t)heads * 128 || ld_out < (int64_t)heads * 128) return RPTC_ERR_SHAPE;
    if (heads > 4096) return RPTC_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(signs_in) & 15) || (ld_q % 8) ||
        (ld_out % 8))
        return RPTC_ERR_ALIGN;
    if (int64_t need = rptc_attn_decode_kv4_workspace_bytes(cache, heads)) {
        if (!workspace || workspace_bytes < need) return RPTC_ERR_ARG;
        if (reinterpret_cast<uintptr_t>(workspace) & 255) return RPTC_ERR_ALIGN;
    }
    if (int e = rptc_check_device()) return e;
    AttnKv4Params p;
    p.q = static_cast<const __half *>(q), p.ld_q = ld_q, p.pos = pos;
    p.k = static_cast<const uint8_t *>(cache->k), p.v = static_cast<const uint8_t *>(cache->v);
    p.k_scales = static_cast<const __half2 *>(cache->k_scales), p.v_scales = static_cast<const __half2 *>(cache->v_scales);
    p.out = static_cast<__half *>(out), p.ld_out = ld_out, p.max_pos = cache->max_pos;
    p.hq = heads, p.hkv = cache->kv_heads, p.scale = scale;
    p.signs_in = static_cast<const __half *>(signs_in);
    p.status = device_status_word();
    if (!p.status) return RPTC_ERR_CUDA;
    return launch(attn_kv4_kernel, dim3((unsigned)heads, (unsigned)cache->rows), dim3(128), 0, static_cast<cudaStream_t>(stream), p);
}
