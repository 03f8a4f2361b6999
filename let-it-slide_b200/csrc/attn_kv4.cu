// Single-query attention over a KV cache in 4 bits (rptc_kv_cache, bits = 4).  No reference counterpart.
//
//   s_j = scale q . k_j,  o = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - m);   k = min + scale_g * code in groups g of 32 values, v alike
//
// The cache is read once, 160 bytes per position and kv head, for up to eight q heads of its group at a time.  A warp takes tiles of 32 positions through a
// private ring of asynchronous copies and multiplies the codes as they are on mma.sync (m16n8k16, fp32 accumulation):
//   scores   A = codes of 16 positions x 16 dims, B = q (column = q head).  A nibble put into the low bits of an fp16 is the number code * 2^-24, exactly, and one
//            four bits higher 16 times that: two masks and half a shift per register, and q's values in the odd places are divided by 16 beforehand (q is first brought to
//            at most 2 by a power of two, so that this loses nothing above 2^-25 of its largest value).  A group's sum is then scaled in fp32:
//            s = sum_g scale_g sum_g(q code) + min_g sum_g(q), the second sum as one more product, of the stored (scale, minimum) pairs with (0, sum_g(q)) in two
//            fp16 parts.
//   output   A = codes - 8 of 16 dims x 16 positions, B = p_j * scale_g in fp16 (one set per group; transposed from the scores' layout by movmatrix):
//            sum p scale (code - 8) + sum p (min + 8 scale).  Codes counted from the middle, so that what the weights' rounding (2^-11, as that of P in any 16-bit
//            product) is multiplied with is not larger than the values; the second sum is in fp32.  (-8 by a product with a constant operand: 173 us where this takes 160.)
// Weights refer to a running maximum of s + log2(a tile's largest scale): the products p * scale then fit fp16 whatever the scales are (2^11 where the reference was set, and
// it moves only when they may pass 2^15, which their sum shows: no maximum is looked for otherwise; what falls below 2^-14 is 2^-25 of the largest).
// Bound: HBM (160 bytes per position and kv head) with the issue slots close behind, about 350 warp instructions per 16 positions: four rows in flight per scheduler at 128
// registers leave a quarter of the slots empty (a round of 16 tiles is 2900 clocks, 163 thousand of the batch's 232 thousand; where the others go was not measured).  32 rows of 500 to 32768 positions, 8 kv heads: 136 us, 5.0 TB/s; one row of 131072: 43.7 us, 3.8 TB/s; one of 200: 4.6 us.
// Long contexts: all tiles of all rows and heads, laid end to end, are cut into equal ranges, two to an SM, so that rows of different lengths balance; a range's
// part of a row goes to the workspace (fp32) and a second kernel joins the parts.  A warp's ring goes on into the range's next item: its first tiles and its q are on their
// way while the item before is finished (32 rows as above 160 us without, and with a join that looked at every row's heads instead of the ranges' ends).
// Short caches take one CTA per row and head and no second kernel (the rule is at kv4_whole).
#include <type_traits>

#include "fwht.cuh"
#include "kv4.cuh"

namespace rptc {

constexpr int kKv4Warps = 8, kKv4Tile = 32, kKv4Stages = 2;
constexpr uint32_t kKv4StageBytes = 2 * kKv4Tile * (kKv4Codes + kKv4Scales);
constexpr uint32_t kKv4Ring = kKv4Warps * kKv4Stages * kKv4StageBytes, kKv4Merge = kKv4Warps * 8 * 128 * 4, kKv4Smem = kKv4Ring + kKv4Merge + kKv4Warps * 8 * 8;
static_assert(kKv4Stages == 2, "a stage is the other one's next");
constexpr float kKv4Bias = 11.f;

struct AttnKv4Params {
    const __half *q;
    int64_t ld_q;
    const int32_t *pos;
    const uint8_t *k, *v;
    const __half2 *k_scales, *v_scales;
    __half *out;
    int64_t ld_out;
    int32_t max_pos, rows, hkv, group, blocks;       // blocks: of eight q heads in a group
    float scale;                                     // includes log2(e)
    const __half *signs_in;
    float4 *part;                                    // [2 * CTAs][8][32]: a part's sums, not divided
    float2 *part_ml;                                 // [2 * CTAs][8]: its maximum and weights' sum
    unsigned int *status;
};

__device__ __forceinline__ int kv4_context(const AttnKv4Params &p, const int32_t *pos, int row) {
    const int at = pos[row];
    return at >= 0 && at < p.max_pos ? at + 1 : 0;
}
__device__ __forceinline__ int kv4_tiles(int context) { return (context + kKv4Tile - 1) / kKv4Tile; }

// How the work is cut: every row's heads laid end to end, each worth its tiles and kKv4Start for what a CTA does around them (q, the warps' sums).  32 rows of 500 to 32768
// take 139.4 us with 16 of those, 135.5 with 20, 135.8 with 24 and 136.7 with 32; kKv4Least is what a CTA is worth starting for.  In numbers of 32 bits: a call whose full rows
// would pass them is refused (kv4_units; a tile counts once for every eight q heads of its kv head).
constexpr uint32_t kKv4Start = 24, kKv4Least = 16;
__device__ __forceinline__ uint32_t kv4_cost(int tiles) { return tiles ? (uint32_t)tiles + kKv4Start : 0u; }
// A CTA has two ranges, one for each eight of its warps, which share nothing.  (Two CTAs of eight warps on an SM: the one that came first is served first and ends long before
// the other, which is then alone: 48 and 61 thousand clocks over 131072 positions, 58 and 58 so; 32 rows as above 142 us, 136 so.)
struct Kv4Cut {
    uint32_t ctas, per, extra, halves;                    // halves: 1, or 0 where all of a CTA's units are its first range's
    __device__ __forceinline__ uint32_t first(uint32_t cta) const { return (per + (cta < extra ? 1u : 0u)) >> halves; }
    __device__ __forceinline__ uint32_t begin(uint32_t range) const {
        const uint32_t cta = range >> 1;
        return cta * per + min(cta, extra) + ((range & 1) ? first(cta) : 0u);
    }
    __device__ __forceinline__ uint32_t range_of(uint32_t at) const {     // the range that a unit is in
        const uint32_t cta = at < extra * (per + 1) ? at / (per + 1) : extra + (at - extra * (per + 1)) / per;
        return 2 * cta + (at - begin(2 * cta) >= first(cta) ? 1u : 0u);
    }
};
__device__ __forceinline__ Kv4Cut kv4_cut(const AttnKv4Params &p, const int32_t *pos, uint32_t most_ctas, int lane) {
    uint32_t sum = 0;
    for (int r0 = 0; r0 < p.rows; r0 += 32) sum += __reduce_add_sync(0xFFFFFFFFu, r0 + lane < p.rows ? kv4_cost(kv4_tiles(kv4_context(p, pos, r0 + lane))) : 0u);
    sum *= (uint32_t)(p.hkv * p.blocks);
    const uint32_t worth = max(sum / kKv4Least, 1u);
    Kv4Cut c;
    c.ctas = min(most_ctas, worth);
    c.halves = worth < 2 * most_ctas ? 0u : 1u;              // few: a range to an SM
    c.per = sum / c.ctas, c.extra = sum - c.per * c.ctas;
    return c;
}
// The row, the head and the place in it that lie `at` units on.  A whole warp.
struct Kv4Place {
    int row, head, context;
    uint32_t cost, off;
};
__device__ __forceinline__ Kv4Place kv4_place(const AttnKv4Params &p, const int32_t *pos, uint32_t at, int lane) {
    const uint32_t heads = (uint32_t)(p.hkv * p.blocks);
    uint32_t before = 0;
    Kv4Place f = {};
    for (int r0 = 0; r0 < p.rows; r0 += 32) {
        const int here = r0 + lane < p.rows ? kv4_context(p, pos, r0 + lane) : 0;
        const uint32_t cost = kv4_cost(kv4_tiles(here));
        uint32_t upto = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, (before + upto) * heads > at);
        if (hit) {
            const int from = __ffs(hit) - 1;
            f.row = r0 + from;
            f.context = __shfl_sync(0xFFFFFFFFu, here, from);
            f.cost = __shfl_sync(0xFFFFFFFFu, cost, from);
            const uint32_t in_row = at - (before + __shfl_sync(0xFFFFFFFFu, upto - cost, from)) * heads;
            f.head = (int)(in_row / f.cost), f.off = in_row - (uint32_t)f.head * f.cost;
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return f;
}
// That many units of an item reach so far into its tiles.
__device__ __forceinline__ int kv4_tile_of(uint32_t units) { return (int)max(units, kKv4Start) - (int)kKv4Start; }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Loads from shared memory at a constant distance from an address, which costs no addition.
template <uint32_t OFF>
__device__ __forceinline__ uint4 lds128_at(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(OFF));
    return v;
}
template <uint32_t OFF>
__device__ __forceinline__ uint2 lds64_at(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(OFF));
    return v;
}
template <uint32_t OFF>
__device__ __forceinline__ uint32_t lds32_at(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(v) : "r"(addr), "n"(OFF));
    return v;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A pair of codes less 8 as fp16, in units of 2^-24: those in the low nibbles of the two halves, and 16 times those in the next ones.  Exact.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return half2_as_u32(__hadd2(u32_as_half2(w & 0x000F000Fu), u32_as_half2(0x80088008u))); }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return half2_as_u32(__hadd2(u32_as_half2(w & 0x00F000F0u), u32_as_half2(0x80808080u))); }

// Four neighbouring values of 128 per lane -> the same of the output, after the output projection's input transform where that is asked for.
__device__ __forceinline__ void kv4_store(const AttnKv4Params &p, int row, int head, int lane, float (&o)[4]) {
    if (p.signs_in) {
        const uint2 s = *reinterpret_cast<const uint2 *>(p.signs_in + head * 128 + 4 * lane);
        const float2 s0 = __half22float2(u32_as_half2(s.x)), s1 = __half22float2(u32_as_half2(s.y));
        o[0] *= s0.x, o[1] *= s0.y, o[2] *= s1.x, o[3] *= s1.y;
        const float a = o[0] + o[1], b = o[0] - o[1], c = o[2] + o[3], d = o[2] - o[3];
        o[0] = a + c, o[1] = b + d, o[2] = a - c, o[3] = b - d;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __shfl_xor_sync(0xFFFFFFFFu, o[i], m);
                o[i] = (lane & m) ? x - o[i] : o[i] + x;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= hadamard_norm_dev(128);
    }
    *reinterpret_cast<uint2 *>(p.out + (int64_t)row * p.ld_out + head * 128 + 4 * lane) =
        make_uint2(half2_as_u32(__floats2half2_rn(o[0], o[1])), half2_as_u32(__floats2half2_rn(o[2], o[3])));
}

template <bool WHOLE>
__global__ void __launch_bounds__(32 * kKv4Warps * (WHOLE ? 1 : 2), WHOLE ? 2 : 1) attn_kv4_kernel(const AttnKv4Params p) {
    extern __shared__ __align__(128) unsigned char all_smem[];
    const int tid = threadIdx.x, lane = tid & 31, eight = WHOLE ? 0 : tid >> 8, warp = (tid >> 5) & 7, g = lane >> 2, t = lane & 3;
    unsigned char *smem = all_smem + eight * kKv4Smem;
    auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + eight), "n"(32 * kKv4Warps) : "memory"); };      // the eight warps
    const uint32_t range = 2 * blockIdx.x + eight;
    const uint32_t ring = smem_addr(smem) + (uint32_t)warp * kKv4Stages * kKv4StageBytes;
    float *merge = reinterpret_cast<float *>(smem + kKv4Ring);
    float2 *merge_ml = reinterpret_cast<float2 *>(smem + kKv4Ring + kKv4Merge);
    pdl_wait_prior_grids();
    pdl_allow_next_grid();                           // not before: the join reads pos without waiting for this kernel's end
    const int32_t *pos = after_wait(p.pos);
    const int heads = p.hkv * p.blocks;              // of a row, in the order of the cut
    // ---- a row's head, its tiles t0 .. t1 - 1; `units` of the range are left behind them ----
    int row, head, context, t0, t1;
    uint32_t units = 0;
    if (WHOLE) {
        row = blockIdx.y, head = blockIdx.x;
        context = kv4_context(p, pos, row);
        if (context == 0 && pos[row] != -1 && tid == 0) atomicExch(p.status, kStatusPosition);
        t0 = 0, t1 = kv4_tiles(context);
    } else {
        const Kv4Cut cut = kv4_cut(p, pos, gridDim.x, lane);
        if (blockIdx.x >= cut.ctas) return;
        const uint32_t at = cut.begin(range);
        units = cut.begin(range + 1) - at;
        if (units == 0) return;
        const Kv4Place f = kv4_place(p, pos, at, lane);
        row = f.row, head = f.head, context = f.context;
        const uint32_t here = min(f.cost - f.off, units);
        t0 = kv4_tile_of(f.off), t1 = kv4_tile_of(f.off + here);
        units -= here;
        if (t0 == t1) return;                        // the range ends in front of the first tile
    }
    auto cache_of = [&](int r, int h) { return ((uint32_t)r * p.hkv + h / p.blocks) * (uint32_t)p.max_pos; };      // in positions: as many as device memory holds
    // q of a head's block, as the lanes use it: of head g the values 8 t .. 8 t + 7 of each group, or null
    auto q_of = [&](int r, int h) -> const __half * {
        const int kvh = h / p.blocks, first = (h - kvh * p.blocks) * 8;
        return g < p.group - first ? p.q + (int64_t)r * p.ld_q + (kvh * p.group + first + g) * 128 + 8 * t : nullptr;
    };
    uint4 raw[4];
    {
        const __half *q = q_of(row, head);
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = q ? ld_ordered_u128(q + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
    }
    // The next item's comes by asynchronous copies into what only this warp reads of the merge buffer (a lane its own bytes); a plain load would wait behind all that the rings
    // ask for, some 7000 clocks.
    auto q_lane = [&](int j) { return smem_addr(merge) + 512u * (8 * j + warp) + 16u * lane; };      // its head of the first four warps' sums
    int stage_no = 0;
    for (bool started = false;; started = true) {
        const uint32_t cache_at = cache_of(row, head);
        // ---- what comes next in the range: it begins with an item's first tile, which is fetched under this one's last ----
        int n_row = row, n_head = head + 1, n_context = context, n_t1 = 0;
        if (!WHOLE && units) {
            if (n_head == heads) {
                n_head = n_context = 0;
                for (++n_row; n_row < p.rows; n_row += 32) {      // over rows without positions
                    const int here = n_row + lane < p.rows ? kv4_context(p, pos, n_row + lane) : 0;
                    const unsigned hit = __ballot_sync(0xFFFFFFFFu, here != 0);
                    if (hit) {
                        n_row += __ffs(hit) - 1;
                        n_context = __shfl_sync(0xFFFFFFFFu, here, __ffs(hit) - 1);
                        break;
                    }
                }
            }
            n_t1 = kv4_tile_of(min(kv4_cost(kv4_tiles(n_context)), units));
        }
        // A tile is 320 pieces of 16 bytes, ten of them a lane's.  (Bulk copies by four lanes took about 70 instructions a tile more: they are issued lane by lane.)
        auto fetch = [&](int tile, int stage) {
            const bool next = !WHOLE && tile >= t1;
            if (next) tile = warp + ((tile - t1) & ~(kKv4Warps - 1));
            if (tile < (next ? n_t1 : t1)) {
                const uint32_t dst = ring + (uint32_t)stage * kKv4StageBytes + 16u * lane, first = (uint32_t)tile * kKv4Tile;
                const uint32_t place = (next ? cache_of(n_row, n_head) : cache_at) + first;
                const int n = (next ? n_context : context) - (int)first;
                const uint64_t codes = (uint64_t)place * kKv4Codes + 16 * lane, scales = (uint64_t)(place + lane) * 4;
                const uint8_t *kc = p.k + codes, *vc = p.v + codes;
                const __half2 *ks = p.k_scales + scales, *vs = p.v_scales + scales;
                if (n >= kKv4Tile) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) cp_async16(dst + 512u * i, kc + 512 * i);
                    cp_async16(dst + kKv4Tile * kKv4Codes, ks);
#pragma unroll
                    for (int i = 0; i < 4; ++i) cp_async16(dst + kKv4Tile * (kKv4Codes + kKv4Scales) + 512u * i, vc + 512 * i);
                    cp_async16(dst + kKv4Tile * (2 * kKv4Codes + kKv4Scales), vs);
                } else {                             // no further than the last position
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (8 * i + (lane >> 2) >= n) continue;
                        cp_async16(dst + 512u * i, kc + 512 * i);
                        cp_async16(dst + kKv4Tile * (kKv4Codes + kKv4Scales) + 512u * i, vc + 512 * i);
                    }
                    if (lane < n) {
                        cp_async16(dst + kKv4Tile * kKv4Codes, ks);
                        cp_async16(dst + kKv4Tile * (2 * kKv4Codes + kKv4Scales), vs);
                    }
                }
            }
            cp_async_commit();                       // an empty group when nothing is left keeps the count constant
        };
        if (n_t1) {
            const __half *q = q_of(n_row, n_head);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (q) cp_async16(q_lane(j), q + 32 * j);
        }
        // The ring's next stages: after the first item they are under way, but for those that a short one does not fill.  The second one asks for its tile after q.
        if (!started || t0 + warp >= t1) fetch(t0 + warp, stage_no);
        // ---- q ----
        uint32_t qb[4][4], q_low[2];                 // q_low: (0, sum of q over group t) in two fp16 parts, against (scale, minimum) pairs
        float unit[2];                               // of the q heads 2 t and 2 t + 1, whose scores this lane gets
        {
            float x[4][8], big = 0.f, mine = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unpack8(raw[j], x[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[j][i]));
            }
            big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
            const int e = big > 0.f ? (int)(__float_as_uint(big) >> 23) - 127 : 0;
            const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[j][i] *= down;
                    sum += x[j][i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float odd = (i & 1) ? 0.0625f : 1.f;
                    qb[j][i] = half2_as_u32(__floats2half2_rn(x[j][i] * odd, x[j][i + 4] * odd));
                }
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                mine = j == t ? sum : mine;
            }
            const __half hi = __float2half_rn(mine);
            q_low[0] = half2_as_u32(__halves2half2(__float2half_rn(0.f), hi));
            q_low[1] = half2_as_u32(__halves2half2(__float2half_rn(0.f), __float2half_rn(mine - __half2float(hi))));
            unit[0] = __shfl_sync(0xFFFFFFFFu, up, 8 * t), unit[1] = __shfl_sync(0xFFFFFFFFu, up, 8 * t + 4);
        }
        if (!started || t0 + warp + kKv4Warps >= t1) fetch(t0 + warp + kKv4Warps, stage_no ^ 1);
        // ---- this warp's tiles ----
        float o[8][4] = {}, low[4][2] = {}, l[2] = {0.f, 0.f}, m[2] = {-INFINITY, -INFINITY};
        const int my_row = (g >> 1) + 4 * (g & 1);   // the position of an operand's row g, so that the V operand's rows t and t + 4 are neighbours in the product
        constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;
        constexpr uint32_t kC = kKv4Codes, kS = kKv4Scales, kKs = kKv4Tile * kC, kV = kKs + kKv4Tile * kS, kVs = kV + kKv4Tile * kC;      // in a stage
        const uint32_t k_lane = ring + my_row * kC + 16 * t, s_lane = ring + my_row * kS, v_lane = ring + t * kC + 8 * g;
#pragma unroll 1
        for (int tile = t0 + warp; tile < t1; tile += kKv4Warps) {
            const uint32_t stage = (uint32_t)stage_no * kKv4StageBytes, k_src = k_lane + stage, s_src = s_lane + stage, v_src = v_lane + stage;
            cp_async_wait<kKv4Stages - 1>();
            __syncwarp();                            // the other lanes' pieces
            const int left = context - tile * kKv4Tile;
            float s[2][4];
            auto scores = [&](auto half) {           // of sixteen positions
                constexpr int u = decltype(half)::value;
                const uint4 xa = lds128_at<16 * u * kC>(k_src), xb = lds128_at<(16 * u + 8) * kC>(k_src);
                const uint4 sa = lds128_at<kKs + 16 * u * kS>(s_src), sb = lds128_at<kKs + (16 * u + 8) * kS>(s_src);
                const uint32_t pa = lds32_at<kKs + 16 * u * kS>(s_src + 4 * t), pb = lds32_at<kKs + (16 * u + 8) * kS>(s_src + 4 * t);
                float low_part[4], part[4];
                mma_first(low_part, pa, pb, pa, pb, q_low[0], q_low[1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    const uint32_t wa = j < 2 ? prmt(xa.x, xa.z, sel) : prmt(xa.y, xa.w, sel), wb = j < 2 ? prmt(xb.x, xb.z, sel) : prmt(xb.y, xb.w, sel);
                    float c[4];
                    mma_first(c, wa & kLow, wb & kLow, wa & kHigh, wb & kHigh, qb[j][0], qb[j][1]);
                    mma_16816(c, (wa >> 8) & kLow, (wb >> 8) & kLow, (wa >> 8) & kHigh, (wb >> 8) & kHigh, qb[j][2], qb[j][3]);
                    const float fa = __low2float(u32_as_half2(j == 0 ? sa.x : j == 1 ? sa.y : j == 2 ? sa.z : sa.w));
                    const float fb = __low2float(u32_as_half2(j == 0 ? sb.x : j == 1 ? sb.y : j == 2 ? sb.z : sb.w));
                    part[0] = j ? fmaf(fa, c[0], part[0]) : fa * c[0];
                    part[1] = j ? fmaf(fa, c[1], part[1]) : fa * c[1];
                    part[2] = j ? fmaf(fb, c[2], part[2]) : fb * c[2];
                    part[3] = j ? fmaf(fb, c[3], part[3]) : fb * c[3];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[u][i] = fmaf(part[i], 16777216.f, low_part[i]);      // in units of q's power of two and the scale
            };
            scores(std::integral_constant<int, 0>());
            scores(std::integral_constant<int, 1>());
            if (left < kKv4Tile) {                   // positions behind the last: whatever the ring holds there
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][i] = 16 * u + 8 * (i >> 1) + my_row < left ? s[u][i] : -INFINITY;
            }
            // ---- weights; their reference moves when a product with the tile's largest v scale may pass 2^15 ----
            float big;
            {
                const uint4 r = lds128_at<kVs>(ring + stage + lane * kS);
                const uint32_t b = half2_as_u32(__hmax2(__hmax2(u32_as_half2(r.x), u32_as_half2(r.y)), __hmax2(u32_as_half2(r.z), u32_as_half2(r.w)))) & 0xFFFFu;
                big = fmaxf(__half2float(__ushort_as_half((unsigned short)__reduce_max_sync(0xFFFFFFFFu, lane < left ? b : 0u))), 5.9604644775390625e-8f);
            }
            float w[2][4], sum[2];
            for (bool known = false;; known = true) {
                const float from0 = kKv4Bias - m[0], from1 = kKv4Bias - m[1];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[u][i] = ex2(fmaf(s[u][i], unit[i & 1], (i & 1) ? from1 : from0));
                sum[0] = (w[0][0] + w[0][2]) + (w[1][0] + w[1][2]), sum[1] = (w[0][1] + w[0][3]) + (w[1][1] + w[1][3]);
                if (known || !__any_sync(0xFFFFFFFFu, !(fmaxf(sum[0], sum[1]) * big <= 32768.f))) break;
                const float log_big = lg2(big);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(fmaxf(s[0][c], s[0][2 + c]), fmaxf(s[1][c], s[1][2 + c]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
                    const float to = fmaxf(m[c], fmaf(top, unit[c], log_big)), f = m[c] == -INFINITY ? 0.f : ex2(m[c] - to);
                    m[c] = to;
                    l[c] *= f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i][c] *= f, o[i][2 + c] *= f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) low[j][c] *= f;
                }
            }
            l[0] += sum[0], l[1] += sum[1];
            // ---- what they are multiplied with ----
            auto values = [&](auto half) {           // of sixteen positions
                constexpr int u = decltype(half)::value;
                const float pa0 = w[u][0], pa1 = w[u][1], pb0 = w[u][2], pb1 = w[u][3];
                uint4 sa = lds128_at<kVs + 16 * u * kS>(s_src), sb = lds128_at<kVs + (16 * u + 8) * kS>(s_src);
                if (left < kKv4Tile) {
                    if (16 * u + my_row >= left) sa = make_uint4(0u, 0u, 0u, 0u);
                    if (16 * u + 8 + my_row >= left) sb = make_uint4(0u, 0u, 0u, 0u);
                }
                const uint2 v0 = lds64_at<kV + 16 * u * kC>(v_src), v1 = lds64_at<kV + (16 * u + 4) * kC>(v_src);
                const uint2 v2 = lds64_at<kV + (16 * u + 8) * kC>(v_src), v3 = lds64_at<kV + (16 * u + 12) * kC>(v_src);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 fa = __half22float2(u32_as_half2(j == 0 ? sa.x : j == 1 ? sa.y : j == 2 ? sa.z : sa.w));
                    const float2 fb = __half22float2(u32_as_half2(j == 0 ? sb.x : j == 1 ? sb.y : j == 2 ? sb.z : sb.w));
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    const uint32_t b0 = transpose8(half2_as_u32(__floats2half2_rn(pa0 * fa.x, pa1 * fa.x)));
                    const uint32_t b1 = transpose8(half2_as_u32(__floats2half2_rn(pb0 * fb.x, pb1 * fb.x)));
                    const uint32_t w0 = j < 2 ? prmt(v0.x, v1.x, sel) : prmt(v0.y, v1.y, sel), w1 = j < 2 ? prmt(v2.x, v3.x, sel) : prmt(v2.y, v3.y, sel);
                    mma_16816(o[2 * j], low_codes(w0), high_codes(w0), low_codes(w1), high_codes(w1), b0, b1);
                    mma_16816(o[2 * j + 1], low_codes(w0 >> 8), high_codes(w0 >> 8), low_codes(w1 >> 8), high_codes(w1 >> 8), b0, b1);
                    const float mid_a = fmaf(8.f, fa.x, fa.y), mid_b = fmaf(8.f, fb.x, fb.y);
                    low[j][0] = fmaf(pa0, mid_a, fmaf(pb0, mid_b, low[j][0]));
                    low[j][1] = fmaf(pa1, mid_a, fmaf(pb1, mid_b, low[j][1]));
                }
            };
            values(std::integral_constant<int, 0>());
            values(std::integral_constant<int, 1>());
            __syncwarp();                            // the stage is free
            fetch(tile + kKv4Stages * kKv4Warps, stage_no);
            stage_no ^= 1;
        }
        // ---- the warps' sums into one ----
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[c] += __shfl_xor_sync(0xFFFFFFFFu, l[c], x);
#pragma unroll
                for (int j = 0; j < 4; ++j) low[j][c] += __shfl_xor_sync(0xFFFFFFFFu, low[j][c], x);
            }
        }
        if (n_t1) {
            cp_async_wait<kKv4Stages - 1>();
            const bool there = q_of(n_row, n_head);
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j] = there ? lds128_at<0>(q_lane(j)) : make_uint4(0u, 0u, 0u, 0u);
        }
        const int kvh = head / p.blocks, first = (head - kvh * p.blocks) * 8, in_block = min(8, p.group - first), q_head = kvh * p.group + first;
        meet();                                      // the last item's sums have been taken
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float *dst = merge + (warp * 8 + 2 * t + c) * 128 + 4 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float mid = low[j][c];
                *reinterpret_cast<float4 *>(dst + 32 * j) = make_float4(fmaf(16777216.f, o[2 * j][c], mid), fmaf(1048576.f, o[2 * j][2 + c], mid),
                                                                         fmaf(16777216.f, o[2 * j + 1][c], mid), fmaf(1048576.f, o[2 * j + 1][2 + c], mid));
            }
            if (g == 0) merge_ml[warp * 8 + 2 * t + c] = make_float2(m[c], l[c]);
        }
        meet();
        if (warp < in_block) {                       // a warp per q head
            float2 ml[kKv4Warps];
            float mx = -INFINITY, den = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kKv4Warps; ++w) ml[w] = merge_ml[w * 8 + warp], mx = fmaxf(mx, ml[w].x);
#pragma unroll
            for (int w = 0; w < kKv4Warps; ++w) {
                const float f = ml[w].x == -INFINITY && ml[w].y == 0.f ? 0.f : ex2(ml[w].x - mx);      // a warp without a tile
                const float4 x = *reinterpret_cast<const float4 *>(merge + (w * 8 + warp) * 128 + 4 * lane);
                den = fmaf(ml[w].y, f, den);
                sum[0] = fmaf(x.x, f, sum[0]), sum[1] = fmaf(x.y, f, sum[1]), sum[2] = fmaf(x.z, f, sum[2]), sum[3] = fmaf(x.w, f, sum[3]);
            }
            if (WHOLE || (t0 == 0 && t1 == kv4_tiles(context))) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = context ? sum[i] / den : 0.f;
                kv4_store(p, row, q_head + warp, lane, sum);
            } else {
                const uint32_t slot = (2 * range + (t0 == 0 ? 1 : 0)) * 8 + warp;
                p.part[slot * 32 + lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
                if (lane == 0) p.part_ml[slot] = make_float2(mx, den);
            }
        }
        if (n_t1 == 0) break;
        units -= min(kv4_cost(kv4_tiles(n_context)), units);
        row = n_row, head = n_head, context = n_context, t0 = 0, t1 = n_t1;
    }
}

// Joins the parts that ranges have left of an item, a CTA per q head of it: of each item where there are few, else of the item that a range's end lies in (`by_item`).
// Also writes the zeros of rows without positions.
constexpr int kKv4JoinWarps = 8;
__global__ void __launch_bounds__(32 * kKv4JoinWarps) attn_kv4_join_kernel(const AttnKv4Params p, uint32_t most_ctas, int by_item) {
    __shared__ float4 sums[kKv4JoinWarps][32];
    __shared__ float2 ml[kKv4JoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // pos was there before the first kernel let this one start: where the parts lie is found before the wait.  (A block of the first kernel has all of its SM's registers, so that
    // a CTA here starts when that block has ended, beside what other SMs still do.)
    const int32_t *pos = after_wait(p.pos);
    const int heads = p.hkv * p.blocks;
    const Kv4Cut cut = kv4_cut(p, pos, most_ctas, lane);
    int row = 0, head = 0, tiles = 0;
    uint32_t first_tile = 0;
    if (by_item) {
        row = blockIdx.x / heads, head = blockIdx.x % heads;
        tiles = kv4_tiles(kv4_context(p, pos, row));
        uint32_t before = 0;
        for (int r0 = 0; r0 < row; r0 += 32) before += __reduce_add_sync(0xFFFFFFFFu, r0 + lane < row ? kv4_cost(kv4_tiles(kv4_context(p, pos, r0 + lane))) : 0u);
        first_tile = before * (uint32_t)heads + (uint32_t)head * kv4_cost(tiles) + kKv4Start;
    } else if (blockIdx.x + 1 < 2 * cut.ctas) {
        const uint32_t at = cut.begin(blockIdx.x + 1);
        const Kv4Place f = kv4_place(p, pos, at, lane);
        if (f.off > kKv4Start) row = f.row, head = f.head, tiles = kv4_tiles(f.context), first_tile = at - f.off + kKv4Start;      // else it ends in front of a first tile
    }
    int c0 = 0, c1 = 0;
    if (tiles) c0 = (int)cut.range_of(first_tile), c1 = (int)cut.range_of(first_tile + tiles - 1);
    const int kvh = head / p.blocks, in_group = (head - kvh * p.blocks) * 8 + blockIdx.y, q_head = kvh * p.group + in_group;
    pdl_wait_prior_grids();
    pdl_allow_next_grid();
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (kv4_context(p, pos, r)) continue;
        if (blockIdx.y == 0 && threadIdx.x == 0 && pos[r] != -1) atomicExch(p.status, kStatusPosition);
        float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int h = blockIdx.y * kKv4JoinWarps + warp; h < p.hkv * p.group; h += gridDim.y * kKv4JoinWarps) kv4_store(p, r, h, lane, zero);
    }
    if (c0 == c1 || (!by_item && c0 != (int)blockIdx.x) || in_group >= p.group) return;      // one range had it all; another CTA has it
    const int every = cut.halves ? 1 : 2, parts = (c1 - c0) / every + 1;      // every other range is empty
    const float4 *part = after_wait(p.part);
    const float2 *part_ml = after_wait(p.part_ml);
    float mx = -INFINITY, den = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 a, float4 x) {
        const float to = fmaxf(mx, a.x), f = mx == -INFINITY ? 0.f : ex2(mx - to), g = ex2(a.x - to);
        mx = to;
        den = fmaf(a.y, g, den * f);
        sum.x = fmaf(x.x, g, sum.x * f), sum.y = fmaf(x.y, g, sum.y * f), sum.z = fmaf(x.z, g, sum.z * f), sum.w = fmaf(x.w, g, sum.w * f);
    };
#pragma unroll 4
    for (int k = warp; k < parts; k += kKv4JoinWarps) {
        const int slot = (2 * (c0 + k * every) + (k == 0 ? 1 : 0)) * 8 + (in_group & 7);
        add(__ldcg(part_ml + slot), __ldcg(part + slot * 32 + lane));
    }
    sums[warp][lane] = sum;
    if (lane == 0) ml[warp] = make_float2(mx, den);
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < kKv4JoinWarps; ++w)
        if (w < parts) add(ml[w], sums[w][lane]);
    float out[4] = {sum.x / den, sum.y / den, sum.z / den, sum.w / den};
    kv4_store(p, row, q_head, lane, out);
}

}  // namespace rptc

using namespace rptc;

// A CTA per row and head, or ranges.  Measured on full caches of 8 kv heads: 1024 positions 9.1 against 9.9 us (one row), 9.3 and 16.7 (16), 51 and 87 (148); 2048 positions
// 13.8 against 10.3 (one row), 14.0 and 13.8 (4), 13.9 and 20.8 (16), 83 and 95 (148).  Longer ones go by ranges whatever the rows are, as those may differ in length; what a long cache
// that holds little costs by that (64 heads over 8; a cache of about its contents, and one of 32768): 200 positions 5.3 and 9.2 us (one row), 5.6 and 13.6 (16), 8.0 and 18.3 (32); 2000
// positions 10.8 and 10.8, 14.2 and 22.0, 23.2 and 33.7.
static bool kv4_whole(const rptc_kv_cache &c, int heads) {
    const int64_t items = (int64_t)c.rows * c.kv_heads * ((heads / c.kv_heads + 7) / 8);
    return c.max_pos <= 1024 || (c.max_pos <= 2048 && 4 * items >= num_sms());
}

// What all rows' heads are worth when full, as the cut counts: below 2^48.
static int64_t kv4_units(const rptc_kv_cache &c, int heads) {
    const int64_t items = (int64_t)c.rows * c.kv_heads * ((heads / c.kv_heads + 7) / 8);
    return items * ((c.max_pos + kKv4Tile - 1) / kKv4Tile + kKv4Start);
}

extern "C" int64_t rptc_attn_decode_kv4_workspace_bytes(const rptc_kv_cache *cache, int heads) {
    if (!cache || check_kv_cache(*cache) || cache->bits != 4 || heads <= 0 || kv4_whole(*cache, heads)) return 0;
    return (int64_t)num_sms() * 2 * 2 * 8 * (128 * 4 + 8);
}

extern "C" int rptc_attn_decode_kv4(const void *q, int64_t ld_q, const int32_t *pos, const rptc_kv_cache *cache, void *out, int64_t ld_out, int heads,
                                    float scale, const void *signs_in, void *workspace, int64_t workspace_bytes, rptc_stream_t stream) {
    if (!q || !pos || !cache || !out) return RPTC_ERR_ARG;
    if (int e = check_kv_cache(*cache)) return e;
    if (cache->bits != 4) return RPTC_ERR_UNSUPPORTED;
    if (!(scale > 0.f && scale < 1e30f)) return RPTC_ERR_ARG;
    if (heads <= 0 || heads % cache->kv_heads || ld_q < (int64_t)heads * 128 || ld_out < (int64_t)heads * 128) return RPTC_ERR_SHAPE;
    if (heads > 4096 || (!kv4_whole(*cache, heads) && kv4_units(*cache, heads) >> 32)) return RPTC_ERR_TOO_LARGE;
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
    p.out = static_cast<__half *>(out), p.ld_out = ld_out;
    p.max_pos = (int32_t)cache->max_pos, p.rows = (int32_t)cache->rows, p.hkv = cache->kv_heads;
    p.group = heads / cache->kv_heads, p.blocks = (p.group + 7) / 8;
    p.scale = scale * 1.4426950408889634f;
    p.signs_in = static_cast<const __half *>(signs_in);
    p.status = device_status_word();
    if (!p.status) return RPTC_ERR_CUDA;
    p.part = nullptr, p.part_ml = nullptr;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv4_whole(*cache, heads)) {
        static SmemOptIn opted;
        if (int e = allow_max_smem(attn_kv4_kernel<true>, opted)) return e;
        return launch(attn_kv4_kernel<true>, dim3((unsigned)(p.hkv * p.blocks), (unsigned)p.rows), dim3(32 * kKv4Warps), kKv4Smem, s, p);
    }
    const int64_t ctas = num_sms(), ranges = 2 * ctas;
    p.part = static_cast<float4 *>(workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part + ranges * 2 * 8 * 32);
    static SmemOptIn opted;
    if (int e = allow_max_smem(attn_kv4_kernel<false>, opted)) return e;
    if (int e = launch(attn_kv4_kernel<false>, dim3((unsigned)ctas), dim3(2 * 32 * kKv4Warps), 2 * kKv4Smem, s, p)) return e;
    // the second kernel starts as SMs come free and waits for the first one's sums itself
    const bool before = pdl_enabled();
    rptc_set_pdl(1);
    const int64_t items = (int64_t)p.rows * p.hkv * p.blocks;
    const int e = launch(attn_kv4_join_kernel, dim3((unsigned)(items < ranges ? items : ranges), (unsigned)(p.group < 8 ? p.group : 8)), dim3(32 * kKv4JoinWarps), 0, s, p,
                         (uint32_t)ctas, items < ranges ? 1 : 0);
    rptc_set_pdl(before ? 1 : 0);
    return e;
}
