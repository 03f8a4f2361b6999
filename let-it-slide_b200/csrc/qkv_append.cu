// The output side of a fused qkv layer for tokens of any sequences (output transform, rotary embedding, append to an fp16 or 4-bit
// cache), and the values that a 4-bit cache stands for.  No reference counterpart.
//
//   y = rope(scale signs H x) per head of 128;   a group of 32 values of k or v: scale = (max - min) / 15, code = round((value - min) / scale), in fp32
//
// Bound: HBM by bytes; in fact the issue slots and the SM's load and store pipe, each some 60 % busy: 2048 tokens of 96 heads 30 us where the traffic is 17 (29 to 31 without the transform
// and into an fp16 cache); 16 tokens 2.5 to 3.0 us, a launch.  The values of a cache: 8.1 us for 2048 positions of 32 kv heads, its traffic 6.7.
#include <type_traits>

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
    int32_t chunk, chunks_q, chunks_kv, chunks;      // heads of a warp (even, or eight); warps of a token: for q, for k (and v), all
    int32_t step_tokens, step_parts;
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
    // Everything advances by two heads.  Of an odd number the last is taken by both halves of the warp, which read it before either writes (x itself may be cleared, or be out).
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
        __syncwarp();                                        // all lanes have read what this step writes
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

// Many tokens of an fp16 x: the transform on the tensor core.  A warp takes eight heads of q, k or v of a token at a time.  With the dims' bits split as J = (0, 1, 2),
// i = (3, 4, 5, 6), H128 = H8(J) x H16(i): for each of the eight J one product H16 X_J (m16n8k16, column = head, the signs exact and the sums in fp32), and H8 as
// additions in a lane, which has the same rows of all eight.  What a lane then holds of its two heads, 2 t and 2 t + 1, are the dims 8 g .. 8 g + 7 and those 64 on: the
// rotation's partner is its own, and a group of 32 is four lanes', of which each ends up with one (head, half) of the four that they share, works out
// its scale and hands it out.
template <int BITS>
__global__ void __launch_bounds__(256, 2) qkv_append_heads_kernel(const AppendParams p) {
    pdl_allow_next_grid();
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // Pieces of work are eight heads of a token; `step` pieces on, so many tokens and parts on (every warp gets q, k and v in turn: they take unequal times).
    const int64_t piece = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    int64_t token = piece / p.chunks;
    int part = (int)(piece - token * p.chunks);
    if (piece >= (int64_t)p.step_tokens * p.chunks + p.step_parts) return;
    uint32_t a[4];                                           // H16: rows g and g + 8, columns i = t, t + 4 (a0, a1), t + 8, t + 12
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int r = g + 8 * (e & 1), i = t + 8 * (e >> 1);
        a[e] = (__popc(r & i) & 1 ? 0xBC00u : 0x3C00u) | (__popc(r & (i + 4)) & 1 ? 0xBC000000u : 0x3C000000u);
    }
    pdl_wait_prior_grids();
    const int32_t *pos_p = after_wait(p.pos), *slot_p = after_wait(p.slots);
    const __half *x = static_cast<const __half *>(after_wait(p.x)) + 8 * t;
    struct Heads {
        int first, count, base;                              // of q, k or v: the first of eight, how many there are, where they lie in a row
        bool q, v;
    };
    auto heads_of = [&](int part) {
        Heads h;
        h.q = part < p.chunks_q, h.v = part >= p.chunks_q + p.chunks_kv;
        h.first = (part - (h.q ? 0 : h.v ? p.chunks_q + p.chunks_kv : p.chunks_q)) * 8;
        h.count = h.q ? p.hq : p.hkv, h.base = h.q ? 0 : h.v ? p.hq + p.hkv : p.hq;
        return h;
    };
    uint4 raw[4];                                            // dims 8 t .. 8 t + 7, and those 32, 64 and 96 on, of head g: all J of i = t, t + 4, ..
    int next_pos = 0;
    int64_t next_slot = 0;
    Heads next = heads_of(part);
    auto fetch = [&]() {
        const uint4 *src = reinterpret_cast<const uint4 *>(x + token * p.ld_x + (next.base + min(next.first + g, next.count - 1)) * 128);
        raw[0] = src[0], raw[1] = src[4], raw[2] = src[8], raw[3] = src[12];
        next_pos = __ldg(pos_p + token), next_slot = slot_p ? __ldg(slot_p + token) : token;
    };
    if (token < p.tokens) fetch();
    while (token < p.tokens) {
        const Heads mine = next;
        const int pos = next_pos, heads = mine.count, base = mine.base, first = mine.first;
        const int64_t slot = next_slot, here = token;
        const bool is_q = mine.q, is_v = mine.v;
        const bool takes = pos >= 0 && pos < p.max_pos && slot >= 0 && slot < p.rows;      // the same in all lanes
        f32x2 cs[4], sn[4];                                  // of the dims 8 g + 2 w and the next
        if (takes && !is_v) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p.angles + (int64_t)pos * 64 + 8 * g + 2 * w));
                cs[w] = pack2(v.x, v.z), sn[w] = pack2(v.y, v.w);
            }
        }
        uint4 signs[2][2];                                   // of head 2 t + c, half
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                signs[c][half] = p.signs ? __ldg(reinterpret_cast<const uint4 *>(p.signs + (base + min(first + 2 * t + c, heads - 1)) * 128 + 64 * half + 8 * g)) : make_uint4(0u, 0u, 0u, 0u);
        f32x2 y[8][2];                                       // [J][half]: heads 2 t and 2 t + 1
#pragma unroll
        for (int J = 0; J < 8; ++J) {
            const uint32_t sel = (J & 1) ? 0x7632u : 0x5410u;
            uint32_t x[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = J < 2 ? raw[q].x : J < 4 ? raw[q].y : J < 6 ? raw[q].z : raw[q].w;
            float d[4];
            mma_first(d, a[0], a[1], a[2], a[3], __byte_perm(x[0], x[1], sel), __byte_perm(x[2], x[3], sel));
            y[J][0] = pack2(d[0], d[1]), y[J][1] = pack2(d[2], d[3]);
        }
        part += p.step_parts, token += p.step_tokens;
        if (part >= p.chunks) part -= p.chunks, ++token;
        if (token < p.tokens) {
            next = heads_of(part);
            fetch();
        }
        if (!takes) {
            if (pos != -1 && lane == 0) atomicExch(p.status, kStatusPosition);
            continue;
        }
#pragma unroll
        for (int h = 1; h < 8; h <<= 1)
#pragma unroll
            for (int J = 0; J < 8; ++J)
                if (!(J & h))
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const f32x2 u = y[J][half], v = y[J + h][half];
                        y[J][half] = add2(u, v), y[J + h][half] = sub2(u, v);
                    }
        uint32_t o[2][2][4];                                 // [head][half][w]: fp16, dims 64 half + 8 g + 2 w and the next
        const f32x2 scale2 = pack2(p.scale, p.scale);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                float u0, u1, v0, v1;
                unpack2(mul2(y[2 * w][half], scale2), u0, u1);
                unpack2(mul2(y[2 * w + 1][half], scale2), v0, v1);
                const uint4 s0 = signs[0][half], s1 = signs[1][half];
                o[0][half][w] = half2_as_u32(__floats2half2_rn(u0, v0)) ^ ((w == 0 ? s0.x : w == 1 ? s0.y : w == 2 ? s0.z : s0.w) & 0x80008000u);
                o[1][half][w] = half2_as_u32(__floats2half2_rn(u1, v1)) ^ ((w == 0 ? s1.x : w == 1 ? s1.y : w == 2 ? s1.z : s1.w) & 0x80008000u);
            }
        if (!is_v) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float2 f = __half22float2(u32_as_half2(o[c][0][w])), s = __half22float2(u32_as_half2(o[c][1][w]));
                    const f32x2 u = pack2(f.x, f.y), v = pack2(s.x, s.y);
                    float m0, m1;
                    unpack2(sub2(mul2(u, cs[w]), mul2(v, sn[w])), m0, m1);
                    o[c][0][w] = half2_as_u32(__floats2half2_rn(m0, m1));
                    unpack2(add2(mul2(v, cs[w]), mul2(u, sn[w])), m0, m1);
                    o[c][1][w] = half2_as_u32(__floats2half2_rn(m0, m1));
                }
        }
        const bool there[2] = {first + 2 * t < heads, first + 2 * t + 1 < heads};
        if (is_q || p.out_kv) {
            __half *dst = p.out + here * p.ld_out + (base + first + 2 * t) * 128 + 8 * g;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (there[c]) {
                    *reinterpret_cast<uint4 *>(dst + 128 * c) = make_uint4(o[c][0][0], o[c][0][1], o[c][0][2], o[c][0][3]);
                    *reinterpret_cast<uint4 *>(dst + 128 * c + 64) = make_uint4(o[c][1][0], o[c][1][1], o[c][1][2], o[c][1][3]);
                }
        }
        if (is_q) continue;
        if (BITS == 16) {
            uint8_t *dst = (is_v ? p.v : p.k) + ((slot * p.max_pos + pos) * p.hkv + first + 2 * t) * 256 + 16 * g;
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (there[c]) {
                    *reinterpret_cast<uint4 *>(dst + 256 * c) = make_uint4(o[c][0][0], o[c][0][1], o[c][0][2], o[c][0][3]);
                    *reinterpret_cast<uint4 *>(dst + 256 * c + 128) = make_uint4(o[c][1][0], o[c][1][1], o[c][1][2], o[c][1][3]);
                }
            continue;
        }
        // (largest, minus the smallest) of the lane's eight values of a (head, half), then of the four lanes': they halve what they look at twice
        uint32_t m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t(&v)[4] = o[e >> 1][e & 1];
            const uint32_t most = half2_as_u32(__hmax2_nan(__hmax2_nan(u32_as_half2(v[0]), u32_as_half2(v[1])), __hmax2_nan(u32_as_half2(v[2]), u32_as_half2(v[3]))));
            const uint32_t least = half2_as_u32(__hmin2_nan(__hmin2_nan(u32_as_half2(v[0]), u32_as_half2(v[1])), __hmin2_nan(u32_as_half2(v[2]), u32_as_half2(v[3])))) ^ 0x80008000u;
            m[e] = half2_as_u32(__hmax2_nan(u32_as_half2(__byte_perm(most, least, 0x5410)), u32_as_half2(__byte_perm(most, least, 0x7632))));
        }
#pragma unroll
        for (int h = 2; h > 0; h >>= 1) {
            const bool up = g & h;
#pragma unroll
            for (int e = 0; e < h; ++e) {
                const uint32_t keep = up ? m[e + h] : m[e], give = up ? m[e] : m[e + h];
                m[e] = half2_as_u32(__hmax2_nan(u32_as_half2(keep), u32_as_half2(__shfl_xor_sync(0xFFFFFFFFu, give, 4 * h))));
            }
        }
        const float2 ends = __half22float2(u32_as_half2(m[0]));      // of head 2 t + (g & 3) / 2, group 2 (g & 1) + g / 4
        float inv;
        const uint32_t scale_min = half2_as_u32(kv4_scale(-ends.y, ends.x, inv));
        const int64_t at = (slot * p.hkv + first + 2 * t) * p.max_pos + pos;
        if (first + 2 * t + ((g >> 1) & 1) < heads)
            reinterpret_cast<uint32_t *>(is_v ? p.v_scales : p.k_scales)[(at + ((g >> 1) & 1) * p.max_pos) * 4 + 2 * (g & 1) + (g >> 2)] = scale_min;
        auto codes = [&](auto small) {
            constexpr bool kSmall = decltype(small)::value;
            uint8_t *dst = (is_v ? p.v : p.k) + at * kKv4Codes + 8 * (2 * (g & 3) + (g >> 2));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t n[2][2];                            // [half]: dims 8 g .. 8 g + 3, the next four
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int from = ((g & 4) | (2 * c + half)) * 4 + t;
                    const float2 sm = __half22float2(u32_as_half2(__shfl_sync(0xFFFFFFFFu, scale_min, from)));
                    const float by = __shfl_sync(0xFFFFFFFFu, inv, from);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 u = __half22float2(u32_as_half2(o[c][half][2 * e])), v = __half22float2(u32_as_half2(o[c][half][2 * e + 1]));
                        n[half][e] = kv4_code(u.x, sm.y, sm.x, by, kSmall) + 16u * kv4_code(u.y, sm.y, sm.x, by, kSmall) + 256u * kv4_code(v.x, sm.y, sm.x, by, kSmall) +
                                     4096u * kv4_code(v.y, sm.y, sm.x, by, kSmall);
                    }
                }
                // four dims of all four groups: those of groups 0 and 2 are in one lane, of 1 and 3 in the lane 16 on
                const uint32_t w0 = __byte_perm(n[0][0], n[1][0], 0x5410), w1 = __byte_perm(n[0][1], n[1][1], 0x5410);
                const uint32_t keep = g < 4 ? w0 : w1, got = __shfl_xor_sync(0xFFFFFFFFu, g < 4 ? w1 : w0, 16), even = g < 4 ? keep : got, odd = g < 4 ? got : keep;
                if (there[c]) *reinterpret_cast<uint2 *>(dst + c * p.max_pos * kKv4Codes) = make_uint2(__byte_perm(even, odd, 0x5410), __byte_perm(even, odd, 0x7632));
            }
        };
        const float step = __low2float(u32_as_half2(scale_min));
        if (__any_sync(0xFFFFFFFFu, step > 0.f && step < kKv4Exact)) codes(std::true_type());
        else codes(std::false_type());
    }
}

template <bool F32, bool TRANSFORM>
static int launch_append(const AppendParams &p, int bits, cudaStream_t s) {
    const dim3 grid((unsigned)p.tokens, (unsigned)((p.chunks + 7) / 8));
    return bits == 4 ? launch(qkv_append_kernel<F32, TRANSFORM, 4>, grid, dim3(256), 0, s, p) : launch(qkv_append_kernel<F32, TRANSFORM, 16>, grid, dim3(256), 0, s, p);
}

// Eight lanes take a position of one kv head: a lane's eight bytes of codes are four values of each group.  There are CTAs for all positions of the rows, whatever they hold: 100 positions
// of 32 rows and 8 kv heads take 4.5 us in a cache of 128, 18 in one of 1024, 544 in one of 32768.
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
    const int pos = blockIdx.x * 32 + (threadIdx.x >> 3);      // the grid covers all positions of a row
    if (pos >= n) return;
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
    // Eight heads at a time where there is work for all SMs and the eights are at least half full (heads of q and of k, fp16; two heads a warp and eight): 2048 tokens of (32, 32)
    // 38 and 30 us, of (64, 8) 29 and 21, of (16, 2) 12.2 and 10.4, of (8, 1) 9.0 and 9.2; 64 of (32, 32) 3.7 and 3.8, of (16, 2) 2.8 and 3.9.
    const int64_t heads = p.hq + 2 * (int64_t)p.hkv, eights = (p.hq + 7) / 8 + 2 * (int64_t)((p.hkv + 7) / 8);
    if (!a->x_is_f32 && a->transform && p.tokens * heads >= 64 * 96 && 4 * eights <= heads) {
        p.chunk = 8;
        p.chunks_q = (p.hq + 7) / 8, p.chunks_kv = (p.hkv + 7) / 8, p.chunks = (int)eights;
        const int64_t pieces = p.tokens * p.chunks, warps = 16 * (int64_t)num_sms();
        int64_t ctas = (pieces + 7) / 8, step = 8 * ctas;
        if (pieces > warps) {                                // a step past the q heads and without a common divisor with the parts
            ctas = warps / 8;
            int on = p.chunks_q + 1;
            auto divisor = [](int a, int b) {
                while (b) {
                    const int r = a % b;
                    a = b, b = r;
                }
                return a;
            };
            while (divisor(on, p.chunks) != 1) ++on;
            step = (warps - on) / p.chunks * p.chunks + on;
        }
        p.step_tokens = (int32_t)(step / p.chunks), p.step_parts = (int32_t)(step % p.chunks);
        return c.bits == 4 ? launch(qkv_append_heads_kernel<4>, dim3((unsigned)ctas), dim3(256), 0, s, p)
                           : launch(qkv_append_heads_kernel<16>, dim3((unsigned)ctas), dim3(256), 0, s, p);
    }
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
