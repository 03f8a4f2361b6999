// Causal attention of packed prompts.  No reference counterpart.
#include <cuda_bf16.h>

#include "common.cuh"

namespace rptc {

struct PromptParams {
    const uint16_t *q, *k, *v;
    uint16_t *out;
    const int32_t *starts, *kv_first, *kv_len;
    int64_t tokens, kv_tokens;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    int32_t sequences, group, d;
    float scale;                     // includes log2(e)
    unsigned int *status;
};

template <bool BF16>
__device__ __forceinline__ float load16(const uint16_t *p) {
    return BF16 ? __bfloat162float(__ushort_as_bfloat16(*p)) : __half2float(__ushort_as_half(*p));
}

// What a sequence has: queries q0 .. q0 + n - 1, keys k0 .. k0 + m - 1, clamped to the tensors.
struct Sequence {
    int q0, n, k0, m;
};
__device__ __forceinline__ Sequence sequence(const PromptParams &p, int s) {
    const int a = __ldg(p.starts + s), b = __ldg(p.starts + s + 1);
    const int k0 = p.kv_first ? __ldg(p.kv_first + s) : a, m = p.kv_len ? __ldg(p.kv_len + s) : b - a;
    Sequence r;
    r.q0 = min(max(a, 0), (int)p.tokens);
    r.n = min(max(b, r.q0), (int)p.tokens) - r.q0;
    r.k0 = min(max(k0, 0), (int)p.kv_tokens);
    r.m = min(max(m, 0), (int)p.kv_tokens - r.k0);
    if (r.q0 != a || r.n != b - a || r.k0 != k0 || r.m != m) atomicExch(p.status, kStatusPosition);
    return r;
}

// A warp per query and head.
template <bool BF16>
__global__ void __launch_bounds__(128) attn_prompt_kernel(const PromptParams p) {
    pdl_allow_next_grid();
    pdl_wait_prior_grids();
    const int s = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 31;
    const Sequence seq = sequence(p, s);
    const int per = p.d / 32;
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 5); i < seq.n; i += gridDim.x * 4) {
        float q[4], acc[4] = {}, m = -INFINITY, l = 0.f;
        const uint16_t *qp = p.q + (int64_t)(seq.q0 + i) * p.q_row + head * p.q_head + lane;
        for (int e = 0; e < 4; ++e) q[e] = e < per ? load16<BF16>(qp + 32 * e) * p.scale : 0.f;
        const int seen = seq.m - seq.n + 1 + i;
        for (int j = 0; j < seen; ++j) {
            const uint16_t *kp = p.k + (int64_t)(seq.k0 + j) * p.k_row + (head / p.group) * p.k_head + lane;
            const uint16_t *vp = p.v + (int64_t)(seq.k0 + j) * p.v_row + (head / p.group) * p.v_head + lane;
            float x = 0.f;
            for (int e = 0; e < per; ++e) x = fmaf(q[e], load16<BF16>(kp + 32 * e), x);
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
            const float mn = fmaxf(m, x), f = exp2f(m - mn), w = exp2f(x - mn);
            m = mn;
            l = l * f + w;
            for (int e = 0; e < per; ++e) acc[e] = fmaf(w, load16<BF16>(vp + 32 * e), acc[e] * f);
        }
        uint16_t *op = p.out + (int64_t)(seq.q0 + i) * p.out_row + head * p.out_head + lane;
        for (int e = 0; e < per; ++e) {
            const float o = seen > 0 ? acc[e] / l : 0.f;
            op[32 * e] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(o)) : __half_as_ushort(__float2half_rn(o));
        }
    }
}

}  // namespace rptc

using namespace rptc;

extern "C" int rptc_attn_prompt(const rptc_prompt_attention *a, rptc_stream_t stream) {
    if (!a || !a->q || !a->k || !a->v || !a->out || !a->starts || !a->kv_first != !a->kv_len) return RPTC_ERR_ARG;
    if ((a->dtype != 0 && a->dtype != 1) || !(a->scale > 0.f && a->scale < 1e30f)) return RPTC_ERR_ARG;
    if (a->d != 64 && a->d != 128) return RPTC_ERR_UNSUPPORTED;
    if (a->tokens < 0 || a->kv_tokens < 0 || a->sequences < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads) return RPTC_ERR_SHAPE;
    if (a->tokens > (1 << 24) || a->kv_tokens > (1 << 24) || a->sequences > 65535 || a->heads > 4096) return RPTC_ERR_TOO_LARGE;
    if (!a->kv_first && a->kv_tokens != a->tokens) return RPTC_ERR_SHAPE;
    for (const void *p : {a->q, a->k, a->v, (const void *)a->out})
        if (reinterpret_cast<uintptr_t>(p) & 15) return RPTC_ERR_ALIGN;
    for (int64_t s : {a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head, a->out_row, a->out_head}) {
        if (s < a->d) return RPTC_ERR_SHAPE;
        if (s % 8) return RPTC_ERR_ALIGN;
    }
    if (int e = rptc_check_device()) return e;
    if (a->tokens == 0 || a->sequences == 0) return RPTC_OK;
    PromptParams p;
    p.q = static_cast<const uint16_t *>(a->q), p.k = static_cast<const uint16_t *>(a->k), p.v = static_cast<const uint16_t *>(a->v);
    p.out = static_cast<uint16_t *>(a->out);
    p.starts = a->starts, p.kv_first = a->kv_first, p.kv_len = a->kv_len;
    p.tokens = a->tokens, p.kv_tokens = a->kv_tokens;
    p.q_row = a->q_row, p.q_head = a->q_head, p.k_row = a->k_row, p.k_head = a->k_head;
    p.v_row = a->v_row, p.v_head = a->v_head, p.out_row = a->out_row, p.out_head = a->out_head;
    p.sequences = (int32_t)a->sequences, p.group = a->heads / a->kv_heads, p.d = a->d;
    p.scale = a->scale * 1.4426950408889634f;
    p.status = device_status_word();
    if (!p.status) return RPTC_ERR_CUDA;
    const int64_t per = (a->tokens + 3) / 4;
    const dim3 grid((unsigned)(per < 2048 ? per : 2048), (unsigned)a->heads, (unsigned)a->sequences);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a->dtype ? launch(attn_prompt_kernel<true>, grid, dim3(128), 0, s, p) : launch(attn_prompt_kernel<false>, grid, dim3(128), 0, s, p);
}
