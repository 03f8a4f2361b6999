// Log probabilities of given tokens, the entropy and the largest entries of rows of logits.  No reference counterpart.
//
//   with M = max x:  z = sum exp(x - M),  w = sum exp(x - M) (x - M);   logprob = (x_t - M) - log z,   entropy = log z - w / z
//
// One pass over the row: a thread keeps M, z and w of its own entries, and they meet at the end.  (x - M first and then its multiple of log2(e): x log2(e) would leave
// fp32's range at the lowest values that masks are made of.)  The largest entries need no second pass either: a thread knows its largest entry, the k-th largest of
// those is a lower bound of the k-th largest entry, and only the (at most k, but for ties) threads that reach it have anything to look for: all threads look, at the few vectors
// that such a thread had read together with its largest entry, and at all of its entries where another of them reaches the bound too.  What is found is ranked by
// (value, index).  Where more is found than there is room for, as in a row of equal entries or one with fewer allowed tokens than are asked for, the k largest are taken one by one, a
// pass over the row each (2048 x 32000 in fp16 with ten tokens allowed, the 20 largest: 1085 us).
// Few rows: a cluster of CTAs shares a row, and each one's sums and k largest meet in the first one's shared memory.
// Bound: HBM, with the special-function unit (an exponential per entry) next: 2048 x 32000 in fp16 20.0 us of traffic, 14.6 of exponentials; 27.5 us measured, 33 with the
// largest entry, 39 with the 20 largest (the meetings of a row's threads, while the SM's other rows read on).  1500 x 128001 in fp32: 117 of traffic, 131, 137 and 146.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace rptc {

namespace cg = cooperative_groups;

constexpr int kLogprobRoom = 512, kLogprobTop = 32, kLogprobUnroll = 4, kLogprobMaxCluster = 8;

struct LogprobParams {
    const void *logits;
    int64_t ld;
    const int64_t *targets;
    float *logprob, *entropy, *top;
    int64_t *ids;
    int64_t n;
    int32_t k;
    unsigned int *status;
};

template <int DTYPE>
__device__ __forceinline__ float logit(const void *row, int64_t i) {
    if (DTYPE == 0) return __half2float(static_cast<const __half *>(row)[i]);
    if (DTYPE == 1) return __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[i]);
    return static_cast<const float *>(row)[i];
}
// The entries of sixteen bytes.
template <int DTYPE, int N>
__device__ __forceinline__ void logits_of(const uint4 &v, float (&x)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DTYPE == 0) {
            const float2 f = __half22float2(u32_as_half2(w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        } else if (DTYPE == 1) {
            x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            x[i] = __uint_as_float(w[i]);
        }
    }
}

// The order of the largest entries as whole numbers: larger logits first, equal ones (0 and -0 too) by their index, NaN in front of all.  Never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);             // -0 + 0 is 0
    return x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) { return (uint64_t)order_of(x) << 32 | (0xFFFFFFFFu - i); }
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t up = (uint32_t)(key >> 32);
    return up == 0xFFFFFFFFu ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float((up & 0x80000000u) ? up & 0x7FFFFFFFu : ~up);
}

__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
template <int DTYPE>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    uint32_t d;
    if (DTYPE == 0) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float ex2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeast = -200.f;      // exp(-200) is 0 in 32 bits, and 0 * -200 is 0: what a forbidden token (-inf) adds

// M, z and w of some entries; NaN among them (or +inf) makes all three NaN, -inf alone leaves M at -inf.
struct Tally {
    float M, z, w;
    __device__ __forceinline__ void move(float to) {         // to >= M, or NaN
        if (M == -INFINITY) {
            M = to;
            return;
        }
        const float d = max_nan(M - to, kLeast), f = ex2_fast(d * kLog2e);
        w = f * fmaf(z, d, w);
        z *= f;
        M = to;
    }
    __device__ __forceinline__ void join(Tally o) {
        const float to = max_nan(M, o.M);
        if (to == -INFINITY) return;
        move(to);
        o.move(to);
        z += o.z;
        w += o.w;
    }
};

__device__ __forceinline__ float warp_max_nan(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
    return x;
}

// A CTA's share of a row: sixteen-byte vectors first .. last - 1, and for the first and last CTA the entries in front of and behind the vectors, one to a thread.
template <int DTYPE>
struct Share {
    static constexpr int kPer = DTYPE == 2 ? 4 : 8;
    const char *row, *vectors;
    int64_t n;
    int32_t head, tail, first, last;                         // entries in front of and behind all vectors
    bool has_head, has_tail;
    __device__ __forceinline__ Share(const void *logits, int64_t r, const LogprobParams &p, int rank, int ranks) {
        constexpr int kSize = DTYPE == 2 ? 4 : 2;
        row = static_cast<const char *>(logits) + r * p.ld * kSize;
        n = p.n;
        const int lead = (int)((0 - reinterpret_cast<uintptr_t>(row)) & 15) / kSize;
        head = (int)min((int64_t)lead, n);
        const int all = (int)((n - head) / kPer);
        tail = (int)(n - head) - all * kPer;
        vectors = row + head * kSize;
        first = (int)((int64_t)all * rank / ranks), last = (int)((int64_t)all * (rank + 1) / ranks);
        has_head = rank == 0, has_tail = rank == ranks - 1;
    }
    __device__ __forceinline__ uint4 vector(int v) const { return __ldg(reinterpret_cast<const uint4 *>(vectors) + v); }
    // the entry outside the vectors that thread t has, or -1
    __device__ __forceinline__ int64_t single(int t) const {
        if (has_head && t < head) return t;
        if (has_tail && t >= 32 && t - 32 < tail) return n - tail + (t - 32);
        return -1;
    }
    __device__ __forceinline__ uint32_t index(int v, int e) const { return (uint32_t)(head + v * kPer + e); }
};

template <int THREADS>
struct LogprobShared {
    static constexpr int kWarps = THREADS / 32;
    Tally tallies[kWarps];
    alignas(16) uint32_t sample[kWarps * 32 + 16];     // the largest of every warp's threads' largest, in the order of the numbers
    int found, chosen, again;
    int at[THREADS], who[THREADS], whole[THREADS];
    alignas(16) uint64_t keys[kLogprobRoom + 8];
    uint64_t best[kLogprobTop], merged[kLogprobMaxCluster * kLogprobTop], round[kWarps];
    Tally tally;
};

// The k largest of the CTA's share, in order (0 where there are fewer), in sh.best.  All threads.
template <int DTYPE, int THREADS>
__device__ void largest_entries(LogprobShared<THREADS> &sh, const Share<DTYPE> &share, float mine, float second, int chunk, int k) {
    constexpr int kPer = Share<DTYPE>::kPer, U = kLogprobUnroll, kWarps = THREADS / 32;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // A bound that at least k threads' largest entries reach: the k-th of a few of every warp, a few more than its part of k, so that it is seldom lower than the k-th of all.
    const int few = min(32, (k + kWarps - 1) / kWarps + 2), samples = few * kWarps;
    const uint32_t own = order_of(mine);
    uint32_t left = own;
    for (int j = 0; j < few; ++j) {
        const uint32_t b = __reduce_max_sync(0xFFFFFFFFu, left);
        if (lane == __ffs(__ballot_sync(0xFFFFFFFFu, left == b)) - 1) {
            left = 0;
            sh.sample[warp * few + j] = b;
        }
    }
    if (t == 0) sh.found = sh.chosen = sh.again = 0;
    sh.at[t] = chunk;
    if (t < k) sh.best[t] = 0;
    if (t >= samples && t < samples + 16) sh.sample[t] = 0;     // to whole rounds of the loop below
    __syncthreads();
    uint32_t bound = 0;                                      // every warp finds it for itself
    for (int i = lane; i < samples; i += 32) {
        const uint32_t x = sh.sample[i];
        int before = 0;
        for (int j = 0; j < samples; j += 16) {
            uint4 y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = *reinterpret_cast<const uint4 *>(sh.sample + j + 4 * e);
#pragma unroll
            for (int e = 0; e < 4; ++e) before += (y[e].x > x) + (y[e].y > x) + (y[e].z > x) + (y[e].w > x);
        }
        if (before < k) bound = bound ? min(bound, x) : x;   // the smallest that fewer than k pass
    }
    bound = __reduce_min_sync(0xFFFFFFFFu, bound ? bound : 0xFFFFFFFFu);
    auto offer = [&](float x, uint32_t i) {
        if (order_of(x) < bound) return;
        const int at = atomicAdd(&sh.found, 1);
        if (at < kLogprobRoom) sh.keys[at] = order_key(x, i);
    };
    if (own >= bound) {
        if (const int64_t s = share.single(t); s >= 0) offer(logit<DTYPE>(share.row, s), (uint32_t)s);
        sh.who[atomicAdd(&sh.chosen, 1)] = t;
        if (order_of(second) >= bound) sh.whole[atomicAdd(&sh.again, 1)] = t;
    }
    __syncthreads();
    auto look = [&](int v) {
        float x[kPer];
        logits_of<DTYPE>(share.vector(v), x);
        float top = x[0];
#pragma unroll
        for (int e = 1; e < kPer; ++e) top = max_nan(top, x[e]);
        if (order_of(top) < bound) return;                   // most have nothing
#pragma unroll
        for (int e = 0; e < kPer; ++e) offer(x[e], share.index(v, e));
    };
    // All threads look at the vectors of those that reach the bound: the few that were read together with the largest
    // entry, and all the others too where one of them reaches it as well.
    const int chosen = sh.chosen, again = sh.again;
    for (int i = t; i < chosen * U; i += THREADS) {
        const int v = sh.at[sh.who[i / U]] + (i % U) * THREADS;
        if (v < share.last) look(v);
    }
    if (again) {
        const int each = (share.last - share.first + THREADS - 1) / THREADS;
        for (int i = t; i < again * each; i += THREADS) {
            const int q = i / each, who = sh.whole[q], v = share.first + who + (i - q * each) * THREADS, from = v - sh.at[who];
            if (v < share.last && (from < 0 || from >= U * THREADS)) look(v);
        }
    }
    __syncthreads();
    const int found = sh.found;
    if (found <= kLogprobRoom) {
        for (int i = t; i < found; i += THREADS) {
            const uint64_t key = sh.keys[i];
            int rank = 0;
            for (int j = 0; j < found; j += 8) {
                ulonglong2 y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = *reinterpret_cast<const ulonglong2 *>(sh.keys + j + 2 * e);
#pragma unroll
                for (int e = 0; e < 4; ++e) rank += (j + 2 * e < found && y[e].x > key) + (j + 2 * e + 1 < found && y[e].y > key);
            }
            if (rank < k) sh.best[rank] = key;
        }
    } else {
        uint64_t last = ~0ull;
        for (int j = 0; j < k; ++j) {                        // one after the other
            uint64_t best = 0;
            auto consider = [&](float x, uint32_t i) {
                const uint64_t key = order_key(x, i);
                if (key < last && key > best) best = key;
            };
            for (int v = share.first + t; v < share.last; v += THREADS) {
                float x[kPer];
                logits_of<DTYPE>(share.vector(v), x);
#pragma unroll
                for (int e = 0; e < kPer; ++e) consider(x[e], share.index(v, e));
            }
            const int64_t s = share.single(t);
            if (s >= 0) consider(logit<DTYPE>(share.row, s), (uint32_t)s);
            for (int o = 16; o > 0; o >>= 1) {
                const uint64_t b = __shfl_xor_sync(0xFFFFFFFFu, best, o);
                best = b > best ? b : best;
            }
            __syncthreads();
            if (lane == 0) sh.round[warp] = best;
            __syncthreads();
            for (int i = 0; i < THREADS / 32; ++i) best = sh.round[i] > best ? sh.round[i] : best;
            last = best;
            if (t == 0) sh.best[j] = best;
        }
    }
    __syncthreads();
}

template <int DTYPE, bool CLUSTER, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 5 : 9) token_logprobs_kernel(const LogprobParams p) {
    constexpr int kPer = Share<DTYPE>::kPer, U = kLogprobUnroll, kWarps = THREADS / 32;
    __shared__ LogprobShared<THREADS> sh;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int rank = 0, ranks = 1;
    int64_t r = blockIdx.x;
    if (CLUSTER) {
        ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
        r = blockIdx.x / ranks;
    }
    pdl_allow_next_grid();
    pdl_wait_prior_grids();
    const Share<DTYPE> share(after_wait(p.logits), r, p, rank, ranks);
    int64_t target = -1;
    float target_logit = 0.f;
    if (t == 64 && rank == 0 && p.targets) {                 // its trip to memory under the others'
        target = after_wait(p.targets)[r];
        if (target >= 0 && target < p.n) target_logit = logit<DTYPE>(share.row, target);
    }
    Tally a = {-INFINITY, 0.f, 0.f};
    float largest = -INFINITY, second = -INFINITY;           // of this thread's entries, and of those not read together with it; NaN if any is
    int chunk = share.last;                                  // the first of the vectors read with the largest
    auto add = [&](const float (&x)[kPer], f32x2 &z, f32x2 &w) {
        const f32x2 unit = pack2(kLog2e, kLog2e), from = pack2(-a.M, -a.M);
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
            float lo, hi;
            unpack2(add2(pack2(x[e], x[e + 1]), from), lo, hi);
            const f32x2 d = pack2(max_nan(lo, kLeast), max_nan(hi, kLeast));
            unpack2(mul2(d, unit), lo, hi);
            const f32x2 q = pack2(ex2_fast(lo), ex2_fast(hi));
            z = add2(z, q);
            w = fma2(q, d, w);
        }
    };
    for (int v0 = share.first + t; v0 < share.last; v0 += U * THREADS) {
        uint4 raw[U];
        // a vector that is not there is one of forbidden tokens
        const uint32_t none = DTYPE == 0 ? 0xFC00FC00u : DTYPE == 1 ? 0xFF80FF80u : 0xFF800000u;
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = v0 + u * THREADS < share.last ? share.vector(v0 + u * THREADS) : make_uint4(none, none, none, none);
        float top = -INFINITY;
        if (DTYPE == 2) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[kPer];
                logits_of<DTYPE>(raw[u], x);
#pragma unroll
                for (int e = 0; e < kPer; ++e) top = max_nan(top, x[e]);
            }
        } else {
            uint32_t m = raw[0].x;                           // pairs
#pragma unroll
            for (int u = 0; u < U; ++u) m = max_pair<DTYPE>(max_pair<DTYPE>(m, max_pair<DTYPE>(raw[u].x, raw[u].y)), max_pair<DTYPE>(raw[u].z, raw[u].w));
            top = DTYPE == 0 ? max_nan(__low2float(u32_as_half2(m)), __high2float(u32_as_half2(m)))
                             : max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
        }
        if (top == -INFINITY) continue;
        if (!(top <= second)) {
            if (!(top <= largest)) {
                second = largest, largest = max_nan(top, largest), chunk = v0;
                a.move(largest);
            } else {
                second = top;
            }
        }
        f32x2 z = pack2(a.z, 0.f), w = pack2(a.w, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[kPer];
            logits_of<DTYPE>(raw[u], x);
            add(x, z, w);
        }
        float lo, hi;
        unpack2(z, lo, hi), a.z = lo + hi;
        unpack2(w, lo, hi), a.w = lo + hi;
    }
    if (const int64_t s = share.single(t); s >= 0) {
        const float x = logit<DTYPE>(share.row, s);
        if (!(x == -INFINITY)) {
            if (!(x <= largest)) {
                largest = max_nan(x, largest);
                a.move(largest);
            }
            const float d = max_nan(x - a.M, kLeast), e = ex2_fast(d * kLog2e);
            a.z += e;
            a.w = fmaf(e, d, a.w);
        }
    }
    const float mine = largest;
    const float warp_top = warp_max_nan(a.M);
    if (!(warp_top == -INFINITY)) a.move(warp_top);
    for (int o = 16; o > 0; o >>= 1) a.z += __shfl_xor_sync(0xFFFFFFFFu, a.z, o), a.w += __shfl_xor_sync(0xFFFFFFFFu, a.w, o);
    if (lane == 0) sh.tallies[warp] = a;
    if (p.k > 0) largest_entries<DTYPE, THREADS>(sh, share, mine, second, chunk, p.k);
    else __syncthreads();
    if (warp == 0) {
        a = sh.tallies[lane % kWarps];
#pragma unroll
        for (int o = 1; o < kWarps; o <<= 1) {
            Tally b;
            b.M = __shfl_xor_sync(0xFFFFFFFFu, a.M, o), b.z = __shfl_xor_sync(0xFFFFFFFFu, a.z, o), b.w = __shfl_xor_sync(0xFFFFFFFFu, a.w, o);
            a.join(b);
        }
        if (lane == 0) sh.tally = a;
    }
    if (CLUSTER) {
        cg::this_cluster().sync();
        if (rank == 0) {                                     // the others' sums and largest entries
            for (int i = t; i < ranks * p.k; i += THREADS) sh.merged[i] = cg::this_cluster().map_shared_rank(sh.best, i / p.k)[i % p.k];
            if (t == 0)
                for (int i = 1; i < ranks; ++i) a.join(*cg::this_cluster().map_shared_rank(&sh.tally, i)), sh.tally = a;
            __syncthreads();
            for (int i = t; i < ranks * p.k; i += THREADS) {
                if (sh.merged[i] == 0) continue;
                int at = 0;
                for (int j = 0; j < ranks * p.k; ++j) at += sh.merged[j] > sh.merged[i];
                if (at < p.k) sh.keys[at] = sh.merged[i];
            }
        }
        cg::this_cluster().sync();                           // nobody leaves before its shared memory has been read
        if (rank) return;
    } else {
        __syncthreads();
    }
    const float M = sh.tally.M, log_z = logf(sh.tally.z);
    auto logprob = [&](float x) { return (x - M) - log_z; };
    if (t < p.k) {
        const uint64_t key = CLUSTER ? sh.keys[t] : sh.best[t];
        p.top[r * p.k + t] = logprob(key_logit(key));
        p.ids[r * p.k + t] = 0xFFFFFFFFu - (uint32_t)key;
    }
    if (t == 32 && p.entropy) p.entropy[r] = log_z - sh.tally.w / sh.tally.z;
    if (t == 64 && p.targets) {
        float lp = 0.f;
        if (target >= 0 && target < p.n) {
            lp = logprob(target_logit);
        } else if (target != -1) {
            lp = __uint_as_float(0x7FFFFFFFu);
            atomicExch(p.status, kStatusPosition);
        }
        p.logprob[r] = lp;
    }
}

template <int DTYPE>
static int launch_logprobs(const LogprobParams &p, int64_t rows, int cluster, int threads, cudaStream_t s) {
    if (threads == 128) return launch(token_logprobs_kernel<DTYPE, false, 128>, dim3((unsigned)rows), dim3(128), 0, s, p);
    if (cluster == 1) return launch(token_logprobs_kernel<DTYPE, false, 256>, dim3((unsigned)rows), dim3(256), 0, s, p);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    RPTC_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<DTYPE, true, 256>, p));
    return RPTC_OK;
}

}  // namespace rptc

using namespace rptc;

extern "C" int rptc_token_logprobs(const void *logits, int dtype, int64_t ld, const int64_t *targets, float *logprob, float *entropy, float *top_logprobs,
                                   int64_t *top_ids, int64_t rows, int64_t n, int top, rptc_stream_t stream) {
    if (!logits || dtype < 0 || dtype > 2 || (targets && !logprob) || top < 0 || (top > 0 && (!top_logprobs || !top_ids))) return RPTC_ERR_ARG;
    if (rows < 0 || n <= 0 || top > n || ld < n) return RPTC_ERR_SHAPE;
    if (top > 32 || n > (1 << 24) || rows > (1 << 24)) return RPTC_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return RPTC_ERR_ALIGN;
    if (int e = rptc_check_device()) return e;
    if (rows == 0) return RPTC_OK;
    LogprobParams p = {logits, ld, targets, logprob, entropy, top_logprobs, top_ids, n, top, device_status_word()};
    if (!p.status) return RPTC_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t bytes = n * (dtype == 2 ? 4 : 2);
    // Few rows: up to eight CTAs share one, as long as each has 32 KiB of it (one row of 8192 in fp16: four CTAs 3.8 us, one 2.5; 32000 in fp16: 4.4 and 4.6; 128001 in
    // fp32: eight 6.8, one 15.8; 148 rows of 32000: two 5.7, one 4.9).
    int cluster = 1;
    while (cluster < kLogprobMaxCluster && rows * cluster * 2 <= 2 * num_sms() && bytes >= cluster * 2 * 32768) cluster *= 2;
    // With the largest entries, whose meetings keep a row's threads waiting, rows of fewer threads and more of them on an SM, unless a row alone has to be fast or is long
    // (top 20, 256 and 128 threads: 8000 rows of 1000 in fp16 72 and 39 us, 2048 of 32000 43 and 39, 300 of 32000 11.9 and 11.7, 800 of 128001 57 and 55, in fp32 145 and 164 for
    // 1500; one of 1000 5.4 and 4.8, one of 32000 7.8 and 9.1).
    const int threads = top > 0 && (bytes <= 4096 || (rows >= 2 * (int64_t)num_sms() && bytes <= 256 * 1024)) ? 128 : 256;
    return dtype == 0 ? launch_logprobs<0>(p, rows, cluster, threads, s) : dtype == 1 ? launch_logprobs<1>(p, rows, cluster, threads, s) : launch_logprobs<2>(p, rows, cluster, threads, s);
}
