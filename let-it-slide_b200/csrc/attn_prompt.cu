// Causal attention of packed prompts on the sm_100a tensor cores.  No reference counterpart.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i)   over the keys that query i sees
//
// An item is 256 query rows of one kv head's queries, in two halves of 128: `pack` heads of a group (the largest power of two that divides it) x
// 256 / pack tokens, so that grouped heads of a short prompt fill the tensor core's 128 rows and share the keys' tiles.  A CTA takes items one after
// the other.  For each tile of 128 keys and each half:
//   S = Q K^T            tcgen05.mma from shared memory into tensor memory (fp32)
//   P = exp2(S - m)      a softmax thread owns a row: it reads its 128 scores, keeps the running maximum m and sum l in registers (as Milakov and Gimelshein, 2018), and puts P back over S in
//                        16 bits (the one rounding besides the result's: the tensor core multiplies 16-bit operands; l adds the weights up before it)
//   O += P V             tcgen05.mma with P in tensor memory, V in shared memory as it lies (N-major), O in tensor memory (fp32)
// The two halves alternate: the tensor core works on one while the other's softmax runs.  m follows the true maximum with a slack of 2^8: only a larger step
// rescales O and l (by the thread that owns the row; the scores' barrier says that the product before has been added).  fp16 weights are 2^7 for a score of m, 2^15 at
// most: what is below fp16's normal numbers is then 2^-21 of the largest weight, and off by 2^-32 of it (with weights of 1 for m many small ones, as behind a first key that takes
// nearly all, came out as zeros: 60000 of 2^-25.5 count for 0.0013).
// Warps 0-3 and 4-7: softmax and output of the halves; 8: MMAs; 9: TMA loads (ring of key and value tiles); 10: the list of items.
// Masks are applied to tiles that reach beyond a half's first row only.  Value rows behind the last key are zeroed in shared memory: a weight of 0 times whatever
// lies there has to be 0.
// Items go to CTAs longest first, there and back again (the longest of a round meets the shortest of the next): the order is worked out from
// `starts` on the device, by counting items of at least a number of tiles.
// Bound: exponentials and products evenly.  A tile of 128 keys and 256 rows takes 2770 to 3000 clocks: 2048 for its 32768 exponentials on the special-function unit, 2048 for its
// products on the tensor core (each busy 69 % of the time at 8192 tokens), which overlap but for a half's softmax that waits for its own product and next scores, and the softmax warps'
// other work.  How long a clock is, power decides: one prompt of 8192 tokens, 64 heads over 8 of 128, fp16, is 1.32 million clocks; ten calls in a row take 845 us each (1.30 PFLOP/s), a
// second of them 965 to 980 (1.45 GHz at the power cap), and queries of zeros 746.  One of 2048 tokens, 32 heads: 64 thousand clocks, 16 tiles of them 47, the set-up (first scores) 7,
// the last result 2; 36 to 38 us.  24 tokens: 6.6 to 7.1 us.  Heads of 64, whose products are half as long and whose exponentials are not: 32 us for 2048 tokens of 32 heads, 675 for 8192 of 64
// over 8.  Sixteen sequences of 1 to 1021 tokens, 64 heads over 8, with `pack` heads together 77 us; when they took 80, one head at a time took 112.  They are 1072 items: a CTA has
// seven, whose starts and ends do not overlap, and at most 37 tiles where the mean is 31, so that an SM has work for 123 of the 145 thousand clocks.
#include <cuda_bf16.h>

#include "tc_ptx.cuh"

namespace rptc {

constexpr int kPromptThreads = 384, kPromptMmaWarp = 8, kPromptLoadWarp = 9, kPromptListWarp = 10;
// 384 threads are launched with 168 registers each, 64512 in all: the same as 256 with 216 and 128 with 72.
constexpr int kPromptSoftmaxRegs = 216, kPromptOtherRegs = 72;
static_assert(256 * kPromptSoftmaxRegs + 128 * kPromptOtherRegs <= 384 * 168, "registers that the block is launched with");
constexpr int kPromptReaders = 10;                   // warps that take items off the list
constexpr uint32_t kPromptPanel = 128 * 128;         // 128 rows of 64 values
constexpr int kTileKeys = 128;
constexpr float kSlack = 8.f;                        // log2 of how far a score may pass the maximum that its row's weights refer to
constexpr float kHalfBias = 7.f;                     // log2 of an fp16 weight whose score is that maximum
static_assert(kSlack + kHalfBias < 16.f, "the largest weight in fp16");

struct PromptParams {
    uint16_t *out;
    const int32_t *starts, *kv_first, *kv_len;
    int64_t tokens, kv_tokens, out_row, out_head;
    int32_t sequences, group, pack, kv_heads, wide;      // wide: rows and heads of out on 32-byte boundaries
    float scale;                                     // includes log2(e)
    unsigned int *status;
};

// What a sequence has: queries q0 .. q0 + n - 1, keys k0 .. k0 + m - 1, clamped to the tensors.
struct Sequence {
    int q0, n, k0, m;
};
__device__ __forceinline__ Sequence sequence(const PromptParams &p, int s) {
    const int a = p.starts[s], b = p.starts[s + 1];
    const int k0 = p.kv_first ? p.kv_first[s] : a, m = p.kv_len ? p.kv_len[s] : b - a;
    Sequence r;
    r.q0 = min(max(a, 0), (int)p.tokens);
    r.n = min(max(b, r.q0), (int)p.tokens) - r.q0;
    r.k0 = min(max(k0, 0), (int)p.kv_tokens);
    r.m = min(max(m, 0), (int)p.kv_tokens - r.k0);
    if (r.q0 != a || r.n != b - a || r.k0 != k0 || r.m != m) atomicExch(p.status, kStatusPosition);
    return r;
}
// How many items of a sequence, of 2^shift tokens each, take at least c tiles of keys (its last ones; all take one).
__device__ __forceinline__ int items_of(const Sequence &s, int shift, int c) {
    const int all = (s.n + (1 << shift) - 1) >> shift;
    if (c <= 1 || all == 0) return all;
    const int reach = kTileKeys * (c - 1);           // an item takes c tiles when its last query sees more keys than these
    if (s.m <= reach) return 0;
    const int first = max(0, reach - (s.m - s.n)) >> shift;
    return all - min(first, all - 1);
}

struct PromptItem {
    int32_t go, head, kv_head, token, tokens, k0, keys, seen, tiles0, tiles1;      // seen: index of the last key that the item's first query sees
    int32_t pad[2];
};

// The items in their order, by one warp.  A lane holds sequence number `lane`; those from 32 on are read again whenever they are counted.  Of one sequence alone, which all
// lanes hold, the order is the reverse of its rows.  Items are asked for in rising order: a search goes on where the last one ended.
struct ItemList {
    const PromptParams &p;
    int lane, shift, groups, most, all = 0;          // most: tiles of the longest item; all: items of a group of heads
    uint32_t total;
    Sequence mine;
    int c = 0, before = 0, end = 0, s0 = 0;          // items of c tiles end in front of `end`; `before` are in front of those of c tiles of sequence s0
    __device__ __forceinline__ ItemList(const PromptParams &params, int l) : p(params), lane(l) {
        shift = 8 - (31 - __clz(p.pack));
        groups = p.kv_heads * p.group / p.pack;
        most = 1;
        if (p.sequences == 1) {
            mine = sequence(p, 0);
            total = (uint32_t)items_of(mine, shift, 1) * groups;
            return;
        }
        mine = {0, 0, 0, 0};
        if (lane < p.sequences) mine = sequence(p, lane);
        most = mine.n > 0 ? (mine.m + kTileKeys - 1) / kTileKeys : 1;
        for (int s = lane + 32; s < p.sequences; s += 32)
            if (const Sequence q = sequence(p, s); q.n > 0) most = max(most, (q.m + kTileKeys - 1) / kTileKeys);
        most = max(1, __reduce_max_sync(0xFFFFFFFFu, most));
        all = count(1);
        total = (uint32_t)all * groups;              // at most 2^28 for the rows and 2^28 for the sequences
    }
    __device__ __forceinline__ int count(int tiles) const {                          // items of at least so many
        int n = items_of(mine, shift, tiles);
        for (int s = lane + 32; s < p.sequences; s += 32) n += items_of(sequence(p, s), shift, tiles);
        return __reduce_add_sync(0xFFFFFFFFu, n);
    }
    __device__ __forceinline__ PromptItem item(uint32_t index) {
        const int per_item = 1 << shift, rank = (int)(index / (uint32_t)groups), heads = (int)(index - (uint32_t)rank * groups);
        Sequence q = mine;
        int j = items_of(mine, shift, 1) - 1 - rank, found = 1;
        if (p.sequences > 1) {
            found = 0;
            if (rank >= end) {                       // the largest c of which there are more than `rank`
                int hi = most;
                c = 1, end = all;
                while (c < hi) {
                    const int mid = c + (hi - c + 1) / 2, n = count(mid);
                    if (n > rank) c = mid, end = n;
                    else hi = mid - 1;
                }
                before = count(c + 1), s0 = 0;
            }
            for (; s0 < p.sequences; s0 += 32) {
                if (s0 > 0) q = s0 + lane < p.sequences ? sequence(p, s0 + lane) : Sequence{0, 0, 0, 0};
                const int from = items_of(q, shift, c), here = from - items_of(q, shift, c + 1), left = rank - before;
                int upto = here;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                    if (lane >= o) upto += v;
                }
                const unsigned hit = __ballot_sync(0xFFFFFFFFu, left < upto);
                if (hit == 0) {
                    before += __shfl_sync(0xFFFFFFFFu, upto, 31);
                    continue;
                }
                const int in = __ffs(hit) - 1;
                j = __shfl_sync(0xFFFFFFFFu, ((q.n + per_item - 1) >> shift) - from + left - (upto - here), in);
                q.q0 = __shfl_sync(0xFFFFFFFFu, q.q0, in), q.n = __shfl_sync(0xFFFFFFFFu, q.n, in);
                q.k0 = __shfl_sync(0xFFFFFFFFu, q.k0, in), q.m = __shfl_sync(0xFFFFFFFFu, q.m, in);
                found = 1;
                break;
            }
        }
        const int splits = p.group / p.pack;
        PromptItem it = {};
        it.go = found;
        it.kv_head = heads / splits;
        it.head = it.kv_head * p.group + (heads - it.kv_head * splits) * p.pack;
        it.token = q.q0 + j * per_item;
        it.tokens = min(per_item, q.n - j * per_item);
        it.k0 = q.k0, it.keys = q.m;
        it.seen = q.m - q.n + j * per_item;
        const int last0 = it.seen + min(it.tokens, per_item / 2), last1 = it.seen + it.tokens;      // keys that a half's last query sees
        it.tiles0 = max(0, (last0 + kTileKeys - 1) / kTileKeys);
        it.tiles1 = it.tokens > per_item / 2 ? max(0, (last1 + kTileKeys - 1) / kTileKeys) : 0;
        return it;
    }
};

// mbar_wait without a call: a function called from here would have to make do with the fewest registers that any warp of the kernel has.
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, unsigned int *status) {
#pragma unroll 1
    for (uint32_t spin = 0; spin < kSpinLimit; ++spin)
        if (mbar_try_wait(bar, parity)) return true;
    atomicExch(status, kStatusWaitExpired);
    return false;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1) attn_prompt_kernel(const PromptParams p, const __grid_constant__ CUtensorMap q_map,
                                                                       const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    constexpr uint32_t kTile = DP * kPromptPanel;    // bytes of a half's queries, of a tile of keys or values
    constexpr int kStages = DP == 2 ? 5 : 8;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base, q_addr = base + 1024u, ring = q_addr + 2 * kTile;
    const uint32_t q_full = bars, q_empty = bars + 8, full = bars + 16, empty = full + 8 * kStages, s_full = empty + 8 * kStages, p_full = s_full + 16,
                   o_full = p_full + 32, item_full = o_full + 16, item_empty = item_full + 16, tail = item_empty + 16, tmem_slot = tail + 8, items = bars + 256;
    if (tid == 0) {
        mbar_init(q_full, 1), mbar_init(q_empty, 1), mbar_init(tail, 1);
        for (int i = 0; i < kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1), mbar_init(o_full + 8 * i, 1);
            mbar_init(p_full + 16 * i, 4), mbar_init(p_full + 16 * i + 8, 4);
            mbar_init(item_full + 8 * i, 1), mbar_init(item_empty + 8 * i, kPromptReaders);
        }
        mbar_fence_init();
    }
    if (warp == kPromptMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    auto set_up = [&]() {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        pdl_allow_next_grid();
    };
    if (warp == kPromptListWarp) {                   // the first item is found while the others set up
        pdl_wait_prior_grids();
        PromptParams q = p;
        q.starts = after_wait(p.starts), q.kv_first = after_wait(p.kv_first), q.kv_len = after_wait(p.kv_len);
        ItemList items_in_order(q, lane);
        const uint32_t total = items_in_order.total;
        PromptItem next = {};
        if (blockIdx.x < total) next = items_in_order.item(blockIdx.x);
        set_up();
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptOtherRegs));
        RingPos list = {0, 0u};
        bool ok = true;
        for (uint32_t round = 0;;) {
            ok = ok && await(item_empty + 8 * list.s, list.phase ^ 1u, p.status);
            if (!__all_sync(0xFFFFFFFFu, ok)) break;
            if (lane == 0) {
                const uint32_t at = items + 64u * list.s;
                const int *w = reinterpret_cast<const int *>(&next);
#pragma unroll
                for (int i = 0; i < 12; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 4u * i), "r"(w[i]) : "memory");
                mbar_arrive(item_full + 8 * list.s);
            }
            __syncwarp();
            list.advance(2);
            if (!next.go) break;                     // the end of the list
            next = {};
            uint32_t index = total;
            while (++round * gridDim.x < total) {    // there and back; the last round may not be full
                index = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                if (index < total) break;
            }
            if (index < total) next = items_in_order.item(index);
        }
    }
    if (warp != kPromptListWarp) set_up();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, lds32(tmem_slot), 0);
    const int rows_per_token = p.pack, half_tokens = 128 / rows_per_token;
    bool ok = true;

    // the next item off the list; false at its end
    RingPos list = {0, 0u};
    auto next_item = [&](PromptItem &it) {
        ok = ok && await(item_full + 8 * list.s, list.phase, p.status);
        if (!__all_sync(0xFFFFFFFFu, ok)) {
            ok = false;
            return false;
        }
        const uint32_t at = items + 64u * list.s;
        const uint4 a = lds128(at), b = lds128(at + 16u), c = lds128(at + 32u);
        it.go = (int)a.x, it.head = (int)a.y, it.kv_head = (int)a.z, it.token = (int)a.w;
        it.tokens = (int)b.x, it.k0 = (int)b.y, it.keys = (int)b.z, it.seen = (int)b.w;
        it.tiles0 = (int)c.x, it.tiles1 = (int)c.y;
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty + 8 * list.s);
        list.advance(2);
        return it.go != 0;
    };

    PromptItem it;
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPromptSoftmaxRegs));
        // ================= softmax and output of one half: a thread owns a row =================
        const int half = warp >> 2, row = (warp & 3) * 32 + lane, my_token = half * half_tokens + row / rows_per_token, my_head = row % rows_per_token;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_tmem = tmem + 128u * half + lanes, o_tmem = tmem + 256u + 128u * half + lanes;
        const uint32_t my_s = s_full + 8 * half, my_p = p_full + 16 * half;
        uint32_t phase = 0u, o_phase = 0u;
        constexpr float kBias = BF16 ? 0.f : kHalfBias;
        while (next_item(it)) {
            const int tiles = half ? it.tiles1 : it.tiles0, first_seen = it.seen + half * half_tokens;
            const int last = min(it.seen + my_token, it.keys - 1);                  // the last key that this row sees
            float m = -INFINITY, l = 0.f;                                           // m: in units of the scores
            for (int i = 0; i < tiles && ok; ++i) {
                ok = await(my_s, phase, p.status);
                phase ^= 1u;
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t s[128], w[32];
                tmem_load64(s_tmem, *reinterpret_cast<uint32_t(*)[64]>(s));
                tmem_load64(s_tmem + 64u, *reinterpret_cast<uint32_t(*)[64]>(s + 64));
                if (i * kTileKeys + kTileKeys - 1 > first_seen || i * kTileKeys + kTileKeys > it.keys) {
                    const int lim = last - i * kTileKeys;
#pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = c <= lim ? s[c] : 0xFF800000u;
                }
                float mx[8];                                                        // (the three-operand maximum takes longer: 2048 tokens, 32 heads 41.9 us, 38.9 so)
#pragma unroll
                for (int c = 0; c < 8; ++c) mx[c] = __uint_as_float(s[c]);
#pragma unroll
                for (int c = 8; c < 128; ++c) mx[c & 7] = fmaxf(mx[c & 7], __uint_as_float(s[c]));
                const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
                if (i == 0) {
                    m = top == -INFINITY ? 0.f : top;                               // a row that sees nothing has weights of 0
                } else {
                    const bool grows = (top - m) * p.scale > kSlack;
                    if (__any_sync(0xFFFFFFFFu, grows)) {
                        const float f = grows ? exp2_fast((m - top) * p.scale) : 1.f;
                        l *= f;
                        m = grows ? top : m;
#pragma unroll 1
                        for (int c = 0; c < DP * 64; c += 32) {
                            uint32_t o[32];
                            tmem_load32(o_tmem + (uint32_t)c, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_store32_begin(o_tmem + (uint32_t)c, o);
                        }
                    }
                }
                const f32x2 scale2 = pack2(p.scale, p.scale), shift2 = pack2(fmaf(-m, p.scale, kBias), fmaf(-m, p.scale, kBias));
                f32x2 sum[4];
#pragma unroll
                for (int c = 0; c < 2; ++c) {                                       // 64 keys: the product takes them while the next are made
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float x, y;
                        unpack2(fma2(pack2(__uint_as_float(s[64 * c + 2 * e]), __uint_as_float(s[64 * c + 2 * e + 1])), scale2, shift2), x, y);
                        x = exp2_fast(x), y = exp2_fast(y);
                        sum[e & 3] = c == 0 && e < 4 ? pack2(x, y) : add2(sum[e & 3], pack2(x, y));
                        w[e] = pack16<BF16>(x, y);
                    }
                    tmem_store32_begin(s_tmem + 32u * c, w);
                    tmem_store_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(my_p + 8 * c);
                }
                float x, y;
                unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), x, y);
                l += x + y;
            }
            if (tiles > 0) {                                                        // the last product has been added
                ok = ok && await(o_full + 8 * half, o_phase, p.status);
                o_phase ^= 1u;
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
            }
            const bool there = my_token < it.tokens;
            const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;               // NaN stays
            uint16_t *out = p.out + (int64_t)(it.token + my_token) * p.out_row + (int64_t)(it.head + my_head) * p.out_head;
            if (p.wide) {
                // 64 columns at a time, 128 bytes of a row.  A store in which every lane has a row of its own touches as many lines as lanes; so four lanes exchange their rows'
                // quarters first, and each store has 128 bytes of eight rows (the sixteen sequences below 80.3 us without, 77.3 so).
                uint16_t *rows[4];
                uint32_t theirs = __ballot_sync(0xFFFFFFFFu, there) >> (lane & 28);
#pragma unroll
                for (int k = 0; k < 4; ++k) rows[k] = reinterpret_cast<uint16_t *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(out), (lane & 28) + k)) + 16 * (lane & 3);
#pragma unroll 1
                for (int c = 0; c < DP * 64; c += 64) {
                    uint32_t o[64], w[4][8];
                    if (tiles > 0) {
                        tmem_load64(o_tmem + (uint32_t)c, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 64; ++e) o[e] = 0u;
                    }
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        const float a = __uint_as_float(o[2 * q]) * inv, b = __uint_as_float(o[2 * q + 1]) * inv;
                        w[q >> 3][q & 7] = inv == 0.f ? 0u : pack16<BF16>(a, b);
                    }
#pragma unroll
                    for (int h = 1; h < 4; h <<= 1) {
                        const bool up = lane & h;
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            if (!(b & h))
#pragma unroll
                                for (int q = 0; q < 8; ++q) {
                                    const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? w[b][q] : w[b + h][q], h);
                                    if (up) w[b][q] = got;
                                    else w[b + h][q] = got;
                                }
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (theirs >> k & 1) st_32_bytes(rows[k] + c, w[k]);
                    __syncwarp();                                                   // what reads tensor memory next is the whole warp
                }
            } else {
                // Rows or heads that lie on 16 bytes only.  The stores are up to a lane; what reads tensor memory is the whole warp, with all of its lanes together.
#pragma unroll 1
                for (int c = 0; c < DP * 64; c += 32) {
                    uint32_t o[32];
                    if (tiles > 0) {
                        tmem_load32(o_tmem + (uint32_t)c, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float a = __uint_as_float(o[e + 2 * q]) * inv, b = __uint_as_float(o[e + 2 * q + 1]) * inv;
                            w[q] = inv == 0.f ? 0u : pack16<BF16>(a, b);
                        }
                        if (there) *reinterpret_cast<uint4 *>(out + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
        }
    } else if (warp == kPromptMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptOtherRegs));
        // ================= MMA issue: the whole warp waits, one lane issues =================
        // One warp for both halves: the order of issue keeps them half a tile apart.  (Two warps: their MMAs interleave, both halves' softmax runs at the same time and
        // the tensor core waits for it.)  What a tile needs besides the weights is waited for under the tile before.
        RingPos pos = {0, 0u};
        uint32_t q_phase = 0u, p_phase[2] = {0u, 0u};
        const uint32_t idesc_s = instr_desc(kTileKeys) | (BF16 ? kInstrBf16 : 0u), idesc_o = instr_desc(DP * 64) | (BF16 ? kInstrBf16 : 0u) | kInstrBMajorN;
        const uint64_t q_desc = umma_desc_sw128(q_addr), k_desc = umma_desc_sw128(ring), v_desc = umma_desc_sw128_mn(ring, kPromptPanel);
        const bool issues = elect_one();
        auto scores = [&](uint32_t half, uint32_t stage) {                          // S = Q K^T
            const uint64_t q = q_desc + half * (kTile >> 4), k = k_desc + stage * (kTile >> 4);
#pragma unroll
            for (uint32_t c = 0; c < 4 * DP; ++c) {
                const uint32_t off = ((c >> 2) * kPromptPanel + (c & 3u) * 32u) >> 4;
                tc_mma_f16(tmem + 128u * half, q + off, k + off, idesc_s, c != 0);
            }
            tc_commit(s_full + 8 * half);
        };
        auto take = [&]() {                                                         // the next stage of the ring, full
            const uint32_t stage = pos.s;
            ok = ok && await(full + 8 * stage, pos.phase, p.status);
            pos.advance(kStages);
            return stage;
        };
        while (next_item(it)) {
            const int tiles = max(it.tiles0, it.tiles1);
            if (tiles == 0) continue;
            ok = ok && await(q_full, q_phase, p.status);
            q_phase ^= 1u;
            uint32_t k_stage = take();
            tc_fence_after();
            if (issues && ok) {
                if (it.tiles0 > 0) scores(0, k_stage);
                if (it.tiles1 > 0) scores(1, k_stage);
                tc_commit(empty + 8 * k_stage);
                if (tiles == 1) tc_commit(q_empty);
            }
            uint32_t v_stage = take();
            if (tiles > 1) k_stage = take();
#pragma unroll 1
            for (int i = 0; i < tiles; ++i) {
                uint32_t v_next = 0, k_next = 0;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    const int mine = h ? it.tiles1 : it.tiles0;
                    if (i < mine) {
                        const uint64_t v = v_desc + v_stage * (kTile >> 4);
                        const uint32_t o_tmem = tmem + 256u + 128u * h, w_tmem = tmem + 128u * h;
                        ok = ok && await(p_full + 16 * h, p_phase[h], p.status);
                        tc_fence_after();
                        if (issues && ok) {                                         // O += P V, 64 keys at a time
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) tc_mma_f16_ta(o_tmem, w_tmem + 8u * c, v + 128u * c, idesc_o, (uint32_t)(i | c) != 0u);
                        }
                        ok = ok && await(p_full + 16 * h + 8, p_phase[h], p.status);
                        p_phase[h] ^= 1u;
                        tc_fence_after();
                        if (issues && ok) {
#pragma unroll
                            for (uint32_t c = 4; c < 8; ++c) tc_mma_f16_ta(o_tmem, w_tmem + 8u * c, v + 128u * c, idesc_o, 1u);
                            // a barrier of its own for the finished sums: the next item's first scores may follow before the softmax warps have looked
                            if (i + 1 < mine) scores(h, k_stage);
                            else tc_commit(o_full + 8 * h);
                        }
                    }
                    if (h == 0 && i + 1 < tiles) {
                        v_next = take();
                        if (i + 2 < tiles) k_next = take();
                    }
                }
                if (issues && ok) {
                    tc_commit(empty + 8 * v_stage);
                    if (i + 1 < tiles) tc_commit(empty + 8 * k_stage);
                    if (i + 2 == tiles) tc_commit(q_empty);
                }
                v_stage = v_next, k_stage = k_next;
            }
        }
    } else if (warp == kPromptLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptOtherRegs));
        // ================= loads =================
        pdl_wait_prior_grids();
        if (lane == 0) tma_prefetch_map(&q_map), tma_prefetch_map(&k_map), tma_prefetch_map(&v_map);
        RingPos pos = {0, 1u};
        uint32_t q_phase = 1u, tail_phase = 0u;
        int64_t loads = 0;
        auto load_tile = [&](const CUtensorMap *map, int tile, uint32_t bar) {
            const bool issues = elect_one();
            ok = ok && await(empty + 8 * pos.s, pos.phase, p.status);
            loads += __all_sync(0xFFFFFFFFu, ok) ? 1 : 0;
            if (issues && ok) {
                mbar_expect_tx(bar, kTile);
#pragma unroll
                for (int d = 0; d < DP; ++d) tma_load_3d(ring + pos.s * kTile + d * kPromptPanel, map, 64 * d, it.kv_head, it.k0 + tile * kTileKeys, bar);
            }
            __syncwarp();
        };
        auto load_values = [&](int tile) {
            const int rows = it.keys - tile * kTileKeys;
            if (rows >= kTileKeys) {
                load_tile(&v_map, tile, full + 8 * pos.s);
            } else {                                                                // the last: rows behind the last key become zeros before anyone reads them
                load_tile(&v_map, tile, tail);
                ok = ok && await(tail, tail_phase, p.status);
                tail_phase ^= 1u;
                for (int x = lane; x < (kTileKeys - rows) * 8 * DP; x += 32) {
                    const int r = rows + x / (8 * DP), piece = x % (8 * DP);
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(ring + pos.s * kTile + (piece >> 3) * kPromptPanel + r * 128u + (piece & 7) * 16u), "r"(0u)
                                 : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one() && ok) mbar_arrive(full + 8 * pos.s);
            }
            pos.advance(kStages);
        };
        auto load_keys = [&](int tile) {
            load_tile(&k_map, tile, full + 8 * pos.s);
            pos.advance(kStages);
        };
        while (next_item(it)) {
            const int tiles = max(it.tiles0, it.tiles1);
            if (tiles == 0) continue;
            {
                const bool issues = elect_one();
                ok = ok && await(q_empty, q_phase, p.status);
                q_phase ^= 1u;
                if (issues && ok) {
                    mbar_expect_tx(q_full, (it.tiles1 > 0 ? 2u : 1u) * kTile);
                    for (int h = 0; h < (it.tiles1 > 0 ? 2 : 1); ++h)
#pragma unroll
                        for (int d = 0; d < DP; ++d)
                            tma_load_3d(q_addr + h * kTile + d * kPromptPanel, &q_map, 64 * d, it.head, it.token + h * half_tokens, q_full);
                }
                __syncwarp();
            }
            load_keys(0);
            for (int i = 0; i < tiles; ++i) {
                load_values(i);
                if (i + 1 < tiles) load_keys(i + 1);
            }
        }
        if (!__all_sync(0xFFFFFFFFu, ok)) {                                         // copies in flight land before the CTA leaves
            for (int i = 0; i < kStages; ++i)
                if (const int64_t n = (loads - i + kStages - 1) / kStages; loads > i) await(full + 8 * i, (uint32_t)(n - 1) & 1u, p.status);
        }
    } else if (warp != kPromptListWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPromptOtherRegs));      // a warp of the third group with nothing to do
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPromptMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

template <int DP, bool BF16>
static int launch_prompt(const PromptParams &p, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s) {
    static SmemOptIn opted;
    auto kern = attn_prompt_kernel<DP, BF16>;
    if (int e = allow_max_smem(kern, opted)) return e;
    return launch(kern, dim3(grid), dim3(kPromptThreads), 2048 + (2 + (DP == 2 ? 5 : 8)) * DP * kPromptPanel, s, p, q, k, v);
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
    if (a->kv_tokens == 0) return RPTC_ERR_SHAPE;
    PromptParams p;
    p.out = static_cast<uint16_t *>(a->out);
    p.starts = a->starts, p.kv_first = a->kv_first, p.kv_len = a->kv_len;
    p.tokens = a->tokens, p.kv_tokens = a->kv_tokens;
    p.out_row = a->out_row, p.out_head = a->out_head;
    p.sequences = (int32_t)a->sequences, p.group = a->heads / a->kv_heads, p.kv_heads = a->kv_heads;
    p.pack = p.group & -p.group;
    if (p.pack > 128) p.pack = 128;
    p.wide = reinterpret_cast<uintptr_t>(a->out) % 32 == 0 && a->out_row % 16 == 0 && a->out_head % 16 == 0;
    p.scale = a->scale * 1.4426950408889634f;
    p.status = device_status_word();
    if (!p.status) return RPTC_ERR_CUDA;
    CUtensorMap q, k, v;
    const bool bf16 = a->dtype == 1;
    if (int e = encode_heads_map(q, a->q, bf16, a->d, a->heads, a->q_head, a->tokens, a->q_row, p.pack, 128 / p.pack)) return e;
    if (int e = encode_heads_map(k, a->k, bf16, a->d, a->kv_heads, a->k_head, a->kv_tokens, a->k_row, 1, kTileKeys)) return e;
    if (int e = encode_heads_map(v, a->v, bf16, a->d, a->kv_heads, a->v_head, a->kv_tokens, a->v_row, 1, kTileKeys)) return e;
    // at most this many items: what `starts` makes of the rows is known on the device alone
    const int64_t most = (a->tokens * p.pack / 256 + a->sequences) * a->kv_heads * (p.group / p.pack);
    const unsigned grid = (unsigned)(most < num_sms() ? most : num_sms());
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->d == 128) return bf16 ? launch_prompt<2, true>(p, q, k, v, grid, s) : launch_prompt<2, false>(p, q, k, v, grid, s);
    return bf16 ? launch_prompt<1, true>(p, q, k, v, grid, s) : launch_prompt<1, false>(p, q, k, v, grid, s);
}
