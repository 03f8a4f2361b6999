// The output side of a fused qkv layer for tokens of any sequences (output transform, rotary embedding, append to an fp16 or 4-bit
// cache), and the values that a 4-bit cache stands for.  No reference counterpart.
//
//   y = rope(scale signs H x) per head of 128;   a group of 32 values of k or v: scale = (max - min) / 15, code = round((value - min) / scale)
//
// Bound: HBM by bytes, the issue slots in fact (shuffles of the transform and the groups' extremes, two heads of a warp at a time): 2048 tokens of 96 heads 38 us where the
// traffic is 17; 16 tokens 2.5 us, a launch.  The values of a cache: 8.1 us for 2048 positions of 32 kv heads, its traffic 6.7.
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
    int32_t chunk, chunks_q, chunks_kv, chunks;      // heads of a warp (even); warps of a token: for q, for k (and v), all
    float scale;                     // includes 1 / sqrt(128) with the transform
    unsigned int *status;
};

// A warp takes `chunk` heads of q, k or v of a token, two at a time: a half-warp holds a head, a lane eight neighbouring values of it, the next pair of heads under way.
// The transform's stages of 8, 16, 32 and 64 and the rotation's partner (64 values on, the lane 8 on) are shuffles; a group of 32 values is four lanes.  Rotation with every
// product rounded, as elementary operations round it: which of two codes a value next to a border gets does not depend on what the compiler fuses.
template <bool F32>
struct EightRaw {
    float4 a, b;                     // fp16: a alone
    uint4 signs;
};
template <bool F32, bool TRANSFORM, int BITS>
__global__ void __launch_bounds__(256) qkv_append_kernel(const AppendParams p) {
    pdl_allow_next_grid();
    const int lane = threadIdx.x & 31, half = lane >> 4, dl = lane & 15;
    const int64_t token = blockIdx.x;
    int part = __shfl_sync(0xFFFFFFFFu, blockIdx.y * 8 + (threadIdx.x >> 5), 0);      // the same in all lanes, and known to be
    if (part >= p.chunks) return;
    const bool is_q = part < p.chunks_q, is_v = part >= p.chunks_q + p.chunks_kv;
    part -= is_q ? 0 : is_v ? p.chunks_q + p.chunks_kv : p.chunks_q;
    const int heads = is_q ? p.hq : p.hkv, base = is_q ? 0 : is_v ? p.hq + p.hkv : p.hq, first = part * p.chunk, end = min(first + p.chunk, heads);
    pdl_wait_prior_grids();
    const int32_t *pos_p = after_wait(p.pos), *slot_p = after_wait(p.slots);
    const int pos = __ldg(pos_p + token);
    const int64_t slot = slot_p ? __ldg(slot_p + token) : token;
    const bool takes = __any_sync(0xFFFFFFFFu, pos >= 0 && pos < p.max_pos && slot >= 0 && slot < p.rows);
    if (!takes && pos != -1 && lane == 0) atomicExch(p.status, kStatusPosition);
    // Everything advances by two heads.  Of an odd number the last is taken by both halves of the warp, which read it before either writes.
    int head = min(first + half, end - 1);
    const char *x = reinterpret_cast<const char *>(p.x) + (token * p.ld_x + (base + head) * 128 + 8 * dl) * (F32 ? 4 : 2);
    const __half *signs = p.signs + (base + head) * 128 + 8 * dl;
    const bool writes = is_q || p.out_kv;
    __half *out = p.out + token * p.ld_out + (base + head) * 128 + 8 * dl;
    auto fetch = [&]() {
        EightRaw<F32> r;
        r.a = reinterpret_cast<const float4 *>(x)[0];
        if (F32) r.b = reinterpret_cast<const float4 *>(x)[1];
        r.signs = make_uint4(0u, 0u, 0u, 0u);
        if (TRANSFORM && p.signs) r.signs = __ldg(reinterpret_cast<const uint4 *>(signs));
        return r;
    };
    EightRaw<F32> next = fetch();
    f32x2 cs[4], sn[4];                                      // sn: minus the sine where the partner is subtracted
    if (takes && !is_v) {
        const float4 *a = reinterpret_cast<const float4 *>(p.angles + (int64_t)pos * 64 + 8 * (dl & 7));
        const float sign = dl < 8 ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = __ldg(a + i);
            cs[i] = pack2(v.x, v.z), sn[i] = pack2(sign * v.y, sign * v.w);
        }
    }
    f32x2 side[4];                                           // +-1: what this lane's value counts in the stages of the transform that are shuffles
#pragma unroll
    for (int m = 0; m < 4; ++m) side[m] = (dl >> m) & 1 ? pack2(-1.f, -1.f) : pack2(1.f, 1.f);
    const int64_t at = BITS == 4 ? (slot * p.hkv + head) * p.max_pos + pos : (slot * p.max_pos + pos) * p.hkv + head;
    uint8_t *cache = (is_v ? p.v : p.k) + (BITS == 4 ? at * kKv4Codes + 4 * (4 * (dl & 3)) + 2 * (dl >> 2) : at * 256 + 16 * dl);
    __half2 *scales = BITS == 4 ? (is_v ? p.v_scales : p.k_scales) + at * 4 + (dl >> 2) : nullptr;
#pragma unroll 1
    for (int left = end - first; left > 0; left -= 2) {
        const EightRaw<F32> raw = next;
        if (F32 && p.clear) {
            float4 *src = reinterpret_cast<float4 *>(const_cast<char *>(x));
            src[0] = src[1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const int step = min(head + 2, end - 1) - head;
        head += step;
        x += step * 128 * (F32 ? 4 : 2);
        signs += step * 128;
        if (left > 2) next = fetch();
        if (!takes) continue;
        f32x2 y[4];
        {
            float v[8];
            if (F32) {
                v[0] = raw.a.x, v[1] = raw.a.y, v[2] = raw.a.z, v[3] = raw.a.w, v[4] = raw.b.x, v[5] = raw.b.y, v[6] = raw.b.z, v[7] = raw.b.w;
            } else {
                unpack8(*reinterpret_cast<const uint4 *>(&raw.a), v);
            }
            if (TRANSFORM) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float a = v[i], b = v[i + 1];
                    y[i / 2] = pack2(a + b, a - b);
                }
                const f32x2 a = add2(y[0], y[1]), b = sub2(y[0], y[1]), c = add2(y[2], y[3]), d = sub2(y[2], y[3]);
                y[0] = add2(a, c), y[1] = add2(b, d), y[2] = sub2(a, c), y[3] = sub2(b, d);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = pack2(v[2 * i], v[2 * i + 1]);
            }
        }
        if (TRANSFORM) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float a, b;
                    unpack2(y[i], a, b);
                    y[i] = fma2(y[i], side[m], pack2(__shfl_xor_sync(0xFFFFFFFFu, a, 1 << m), __shfl_xor_sync(0xFFFFFFFFu, b, 1 << m)));
                }
        }
        const uint32_t bits[4] = {raw.signs.x, raw.signs.y, raw.signs.z, raw.signs.w}, scale = __float_as_uint(p.scale);
        uint32_t o16[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {                        // the layer's fp16 output, then the rotation of q and k
            float a, b;
            unpack2(mul2(y[i], TRANSFORM ? pack2(__uint_as_float(scale ^ ((bits[i] << 16) & 0x80000000u)), __uint_as_float(scale ^ (bits[i] & 0x80000000u)))
                                         : pack2(p.scale, p.scale)), a, b);
            o16[i] = half2_as_u32(__floats2half2_rn(a, b));
            if (!is_v) {
                const float2 f = __half22float2(u32_as_half2(o16[i])), o = __half22float2(u32_as_half2(__shfl_xor_sync(0xFFFFFFFFu, o16[i], 8)));
                unpack2(add2(mul2(pack2(f.x, f.y), cs[i]), mul2(pack2(o.x, o.y), sn[i])), a, b);
                o16[i] = half2_as_u32(__floats2half2_rn(a, b));
            }
        }
        const uint4 whole = make_uint4(o16[0], o16[1], o16[2], o16[3]);
        if (writes) *reinterpret_cast<uint4 *>(out) = whole;
        out += step * 128;
        if (is_q) continue;
        if (BITS == 16) {
            *reinterpret_cast<uint4 *>(cache) = whole;
            cache += step * 256;
        } else {
            float v[8];
            __half2 sm;
            unpack8(whole, v);
            const uint32_t codes = kv4_quantise(v, sm);      // all lanes take part
            unsigned short *c = reinterpret_cast<unsigned short *>(cache);          // pieces 2 (dl % 4) and the next
            c[0] = (unsigned short)codes;
            c[4] = (unsigned short)(codes >> 16);
            if ((dl & 3) == 0) *scales = sm;
            cache += step * p.max_pos * kKv4Codes;
            scales += step * p.max_pos * 4;
        }
    }
}

template <bool F32, bool TRANSFORM>
static int launch_append(const AppendParams &p, int bits, cudaStream_t s) {
    const dim3 grid((unsigned)p.tokens, (unsigned)((p.chunks + 7) / 8));
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
        for (int j = 0; j < 4; j += 2) {                     // two groups at a time: one rounding, that of the fused multiply-add
            const uint32_t scale = __byte_perm(s[j], s[j + 1], 0x5410), least = __byte_perm(s[j], s[j + 1], 0x7632);
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = half2_as_u32(__hfma2(__hsub2(u32_as_half2(((w[j >> 1] >> (4 * i)) & 0x000F000Fu) | 0x64006400u), u32_as_half2(0x64006400u)), u32_as_half2(scale), u32_as_half2(least)));
            *reinterpret_cast<uint2 *>(dst + 32 * j) = make_uint2(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410));
            *reinterpret_cast<uint2 *>(dst + 32 * j + 32) = make_uint2(__byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632));
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
    // A warp's heads share their token's angles and place; where there are few tokens more warps are worth more (2048 tokens of 96 heads: two heads a warp 60 us, four
    // 44, eight 38; 16 tokens 2.5, 3.1 and 4.1).
    const int64_t pairs = a->tokens * ((p.hq + 1) / 2 + 2 * ((p.hkv + 1) / 2));
    p.chunk = pairs >= 4 * 24 * (int64_t)num_sms() ? 8 : pairs >= 2 * 24 * (int64_t)num_sms() ? 4 : 2;
    p.chunks_q = (p.hq + p.chunk - 1) / p.chunk, p.chunks_kv = (p.hkv + p.chunk - 1) / p.chunk;
    p.chunks = p.chunks_q + 2 * p.chunks_kv;
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
