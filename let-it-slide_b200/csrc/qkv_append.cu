// The output side of a fused qkv layer for tokens of any sequences (output transform, rotary embedding, append to an fp16 or 4-bit
// cache), and the values that a 4-bit cache stands for.  No reference counterpart.
#include "fwht.cuh"
#include "kv4.cuh"

namespace rptc {

struct AppendParams {
    const void *x;
    int64_t ld_x;
    const __half *signs;
    const int32_t *slots, *pos;
    const float2 *angles;            // [max_pos][64] cosine, sine
    __half *out;
    int64_t ld_out, tokens;
    uint8_t *k, *v;                  // codes, or fp16 rows
    __half2 *k_scales, *v_scales;
    int64_t rows, max_pos;
    int32_t hq, hkv, clear, out_kv;
    int32_t chunk, chunks;           // heads of a warp (even), warps of a token
    float scale;                     // includes 1 / sqrt(128) with the transform
    unsigned int *status;
};

// A warp takes `chunk` heads of a token, two at a time: a half-warp holds a head, a lane eight neighbouring values of it.  The
// rotation's partner (64 values on) is the lane 8 on, a group of 32 values is four lanes.  Rotation with every product rounded, as elementary operations
// round it: which of two codes a value next to a border gets does not depend on what the compiler fuses.
template <bool F32, bool TRANSFORM, int BITS>
__global__ void __launch_bounds__(256) qkv_append_kernel(const AppendParams p) {
    pdl_allow_next_grid();
    const int lane = threadIdx.x & 31, half = lane >> 4, dl = lane & 15;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t token = w / p.chunks;
    const int first = (int)(w - token * p.chunks) * p.chunk, heads = p.hq + 2 * p.hkv;
    pdl_wait_prior_grids();
    if (token >= p.tokens) return;                           // of a whole warp
    const int32_t *pos_p = after_wait(p.pos), *slot_p = after_wait(p.slots);
    const int pos = __ldg(pos_p + token);
    const int64_t slot = slot_p ? __ldg(slot_p + token) : token;
    const bool takes = pos >= 0 && pos < p.max_pos && slot >= 0 && slot < p.rows;
    if (!takes && pos != -1 && lane == 0) atomicExch(p.status, kStatusPosition);
    float cs[8], sn[8];
    if (takes) {
        const float4 *a = reinterpret_cast<const float4 *>(p.angles + (int64_t)pos * 64 + 8 * (dl & 7));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = __ldg(a + i);
            cs[2 * i] = v.x, sn[2 * i] = v.y, cs[2 * i + 1] = v.z, sn[2 * i + 1] = v.w;
        }
    }
#pragma unroll 2
    for (int h0 = first; h0 < min(first + p.chunk, heads); h0 += 2) {
        const int head = h0 + half;
        const bool there = head < heads;
        float v[8] = {};
        if (F32) {
            if (there) load8_f32(const_cast<float *>(static_cast<const float *>(p.x)) + token * p.ld_x + head * 128 + 8 * dl, v, p.clear);
        } else {
            if (there) load8_f16(static_cast<const __half *>(p.x) + token * p.ld_x + head * 128 + 8 * dl, v);
        }
        if (!takes) continue;
        if (TRANSFORM) {
            float s[8];
            unpack8(raw8_or_ones(p.signs && there ? p.signs + head * 128 + 8 * dl : nullptr), s);
            fwht8(v, 128, nullptr);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __half2float(__float2half_rn(__fmul_rn(v[i] * p.scale, s[i])));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __half2float(__float2half_rn(v[i] * p.scale));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o = __shfl_xor_sync(0xFFFFFFFFu, v[i], 8);
            const float turned = dl < 8 ? __fsub_rn(__fmul_rn(v[i], cs[i]), __fmul_rn(o, sn[i])) : __fadd_rn(__fmul_rn(v[i], cs[i]), __fmul_rn(o, sn[i]));
            if (head < p.hq + p.hkv) v[i] = __half2float(__float2half_rn(turned));
        }
        if (there && (head < p.hq || p.out_kv)) store8_f16(p.out + token * p.ld_out + head * 128 + 8 * dl, v);
        const bool is_v = head >= p.hq + p.hkv, cached = there && head >= p.hq;
        const int kvh = head - p.hq - (is_v ? p.hkv : 0);
        if (BITS == 16) {
            if (cached) store8_f16(reinterpret_cast<__half *>(is_v ? p.v : p.k) + ((slot * p.max_pos + pos) * p.hkv + kvh) * 128 + 8 * dl, v);
        } else {
            __half2 sm;
            const uint32_t codes = kv4_quantise(v, sm);      // all lanes take part
            if (cached) {
                const int64_t at = (slot * p.hkv + kvh) * p.max_pos + pos;
                const int group = dl >> 2, piece = 2 * (dl & 3);
                unsigned short *c = reinterpret_cast<unsigned short *>((is_v ? p.v : p.k) + at * kKv4Codes) + 4 * piece + group;
                c[0] = (unsigned short)codes;
                c[4] = (unsigned short)(codes >> 16);
                if ((dl & 3) == 0) (is_v ? p.v_scales : p.k_scales)[at * 4 + group] = sm;
            }
        }
    }
}

template <bool F32, bool TRANSFORM>
static int launch_append(const AppendParams &p, int bits, cudaStream_t s) {
    const dim3 grid((unsigned)((p.tokens * p.chunks + 7) / 8));
    return bits == 4 ? launch(qkv_append_kernel<F32, TRANSFORM, 4>, grid, dim3(256), 0, s, p) : launch(qkv_append_kernel<F32, TRANSFORM, 16>, grid, dim3(256), 0, s, p);
}

// Eight lanes take a position of one kv head: a lane's eight bytes of codes are four values of each group.
__global__ void __launch_bounds__(256) kv4_values_kernel(const uint8_t *__restrict__ k, const __half2 *__restrict__ k_scales, const uint8_t *__restrict__ v,
                                                         const __half2 *__restrict__ v_scales, const int32_t *__restrict__ count, __half *__restrict__ k_out,
                                                         __half *__restrict__ v_out, int max_pos, int hkv, unsigned int *status) {
    pdl_allow_next_grid();
    pdl_wait_prior_grids();
    const int head = blockIdx.y % hkv, g = threadIdx.x & 7;
    const int64_t row = blockIdx.y / hkv;
    const int n = *after_wait(count + row);
    if (n < 0 || n > max_pos) {
        if (threadIdx.x == 0) atomicExch(status, kStatusPosition);
        return;
    }
    const uint8_t *codes = after_wait(blockIdx.z ? v : k);
    const __half2 *scales = after_wait(blockIdx.z ? v_scales : k_scales);
    __half *out = blockIdx.z ? v_out : k_out;
    for (int pos = blockIdx.x * 32 + (threadIdx.x >> 3); pos < n; pos += gridDim.x * 32) {
        const int64_t at = (int64_t)blockIdx.y * max_pos + pos;
        const uint2 c = *reinterpret_cast<const uint2 *>(codes + at * kKv4Codes + 8 * g);
        const uint4 sm = *reinterpret_cast<const uint4 *>(scales + at * 4);
        const uint32_t w[2] = {c.x, c.y}, s[4] = {sm.x, sm.y, sm.z, sm.w};
        __half *dst = out + ((row * max_pos + pos) * hkv + head) * 128 + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(u32_as_half2(s[j]));
            const uint32_t n4 = w[j >> 1] >> (16 * (j & 1));
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf((float)((n4 >> (4 * i)) & 15u), f.x, f.y);
            *reinterpret_cast<uint2 *>(dst + 32 * j) = make_uint2(half2_as_u32(__floats2half2_rn(o[0], o[1])), half2_as_u32(__floats2half2_rn(o[2], o[3])));
        }
    }
}

}  // namespace rptc

using namespace rptc;

extern "C" int rptc_qkv_append(const rptc_append *a, rptc_stream_t stream) {
    if (!a || !a->x || !a->pos || !a->angles || !a->out) return RPTC_ERR_ARG;
    if (int e = check_kv_cache(a->cache)) return e;
    const rptc_kv_cache &c = a->cache;
    if (a->signs_out && !a->transform) return RPTC_ERR_ARG;
    if (a->clear && !a->x_is_f32) return RPTC_ERR_ARG;
    if (a->heads <= 0 || a->heads % c.kv_heads || a->tokens < 0) return RPTC_ERR_SHAPE;
    if (a->heads > 4096 || a->tokens > (1 << 24)) return RPTC_ERR_TOO_LARGE;
    const int64_t all = (int64_t)(a->heads + 2 * c.kv_heads) * 128;
    if (a->ld_x < all || a->ld_out < (a->out_kv ? all : (int64_t)a->heads * 128)) return RPTC_ERR_SHAPE;
    if (!a->slots && a->tokens > c.rows) return RPTC_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a->x) & 15) || (reinterpret_cast<uintptr_t>(a->out) & 15) || (reinterpret_cast<uintptr_t>(a->signs_out) & 15) ||
        (reinterpret_cast<uintptr_t>(a->angles) & 15) || (a->ld_x % (a->x_is_f32 ? 4 : 8)) || (a->ld_out % 8))
        return RPTC_ERR_ALIGN;
    if (int e = rptc_check_device()) return e;
    if (a->tokens == 0) return RPTC_OK;
    AppendParams p;
    p.x = a->x, p.ld_x = a->ld_x;
    p.signs = static_cast<const __half *>(a->signs_out);
    p.slots = a->slots, p.pos = a->pos;
    p.angles = reinterpret_cast<const float2 *>(a->angles);
    p.out = static_cast<__half *>(a->out), p.ld_out = a->ld_out, p.tokens = a->tokens;
    p.k = static_cast<uint8_t *>(c.k), p.v = static_cast<uint8_t *>(c.v);
    p.k_scales = static_cast<__half2 *>(c.k_scales), p.v_scales = static_cast<__half2 *>(c.v_scales);
    p.rows = c.rows, p.max_pos = c.max_pos;
    p.hq = a->heads, p.hkv = c.kv_heads, p.clear = a->clear, p.out_kv = a->out_kv;
    p.chunk = 2;
    p.chunks = (p.hq + 2 * p.hkv + p.chunk - 1) / p.chunk;
    p.scale = a->transform ? (float)((double)a->scale * 0.08838834764831845) : a->scale;
    p.status = device_status_word();
    if (!p.status) return RPTC_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->x_is_f32) return a->transform ? launch_append<true, true>(p, c.bits, s) : launch_append<true, false>(p, c.bits, s);
    return a->transform ? launch_append<false, true>(p, c.bits, s) : launch_append<false, false>(p, c.bits, s);
}

extern "C" int rptc_kv4_values(const rptc_kv_cache *cache, const int32_t *count, void *k_out, void *v_out, rptc_stream_t stream) {
    if (!cache || !count || !k_out || !v_out) return RPTC_ERR_ARG;
    if (int e = check_kv_cache(*cache)) return e;
    if (cache->bits != 4) return RPTC_ERR_UNSUPPORTED;
    if (cache->rows * cache->kv_heads > 65535) return RPTC_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(k_out) & 15) || (reinterpret_cast<uintptr_t>(v_out) & 15)) return RPTC_ERR_ALIGN;
    if (int e = rptc_check_device()) return e;
    unsigned int *status = device_status_word();
    if (!status) return RPTC_ERR_CUDA;
    const dim3 grid((unsigned)((cache->max_pos + 31) / 32), (unsigned)(cache->rows * cache->kv_heads), 2);
    return launch(kv4_values_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t *>(cache->k),
                  static_cast<const __half2 *>(cache->k_scales), static_cast<const uint8_t *>(cache->v), static_cast<const __half2 *>(cache->v_scales), count,
                  static_cast<__half *>(k_out), static_cast<__half *>(v_out), (int)cache->max_pos, cache->kv_heads, status);
}
