// Log probabilities of given tokens, the entropy and the largest entries of rows of logits.  No reference counterpart.
#include <cuda_bf16.h>

#include "common.cuh"

namespace rptc {

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

// The order of the largest entries as whole numbers: larger logits first, equal ones (0 and -0 too) by their index, NaN in front of all.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.f);             // -0 + 0 is 0
    const uint32_t up = x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)up << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t up = (uint32_t)(key >> 32);
    return up == 0xFFFFFFFFu ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float((up & 0x80000000u) ? up & 0x7FFFFFFFu : ~up);
}

// Running maximum m, z = sum exp(x - m) and w = sum exp(x - m) (x - m).  A forbidden token (-inf) adds nothing; with NaN or +inf z and w become NaN.
struct Tally {
    float m = -INFINITY, z = 0.f, w = 0.f;
    __device__ __forceinline__ void move(float to) {
        if (to == m || m == -INFINITY) {
            m = to;
            return;
        }
        const float d = m - to, f = __expf(d);
        w = f * fmaf(z, f == 0.f ? 0.f : d, w);              // where f is 0, d may be too large for a product
        z *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        if (x == -INFINITY) return;
        if (x > m) move(x);
        const float d = x - m, e = __expf(d);
        z += e;
        w = fmaf(e, e == 0.f ? 0.f : d, w);
    }
    __device__ __forceinline__ void join(Tally o) {
        const float to = fmaxf(m, o.m);
        move(to);
        o.move(to);
        z += o.z;
        w += o.w;
    }
};

template <int DTYPE>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const LogprobParams p) {
    __shared__ Tally tallies[8];
    __shared__ uint64_t keys[8];
    pdl_allow_next_grid();
    pdl_wait_prior_grids();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int64_t r = blockIdx.x;
    const char *row = static_cast<const char *>(after_wait(p.logits)) + r * p.ld * (DTYPE == 2 ? 4 : 2);
    Tally a;
    for (int64_t i = t; i < p.n; i += 256) a.add(logit<DTYPE>(row, i));
    for (int o = 16; o > 0; o >>= 1) {
        Tally b;
        b.m = __shfl_xor_sync(0xFFFFFFFFu, a.m, o), b.z = __shfl_xor_sync(0xFFFFFFFFu, a.z, o), b.w = __shfl_xor_sync(0xFFFFFFFFu, a.w, o);
        a.join(b);
    }
    if (lane == 0) tallies[warp] = a;
    __syncthreads();
    a = tallies[0];
    for (int i = 1; i < 8; ++i) a.join(tallies[i]);
    const float log_z = logf(a.z);
    if (t == 0) {
        if (p.entropy) p.entropy[r] = log_z - a.w / a.z;
        if (p.targets) {
            const int64_t at = after_wait(p.targets)[r];
            float lp = 0.f;
            if (at >= 0 && at < p.n) {
                lp = (logit<DTYPE>(row, at) - a.m) - log_z;
            } else if (at != -1) {
                lp = __uint_as_float(0x7FFFFFFFu);
                atomicExch(p.status, kStatusPosition);
            }
            p.logprob[r] = lp;
        }
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < p.k; ++j) {
        uint64_t best = 0;
        for (int64_t i = t; i < p.n; i += 256) {
            const uint64_t key = order_key(logit<DTYPE>(row, i), (uint32_t)i);
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t b = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            best = b > best ? b : best;
        }
        __syncthreads();
        if (lane == 0) keys[warp] = best;
        __syncthreads();
        for (int i = 0; i < 8; ++i) best = keys[i] > best ? keys[i] : best;
        last = best;
        if (t == 0) {
            p.top[r * p.k + j] = (key_logit(best) - a.m) - log_z;
            p.ids[r * p.k + j] = 0xFFFFFFFFu - (uint32_t)best;
        }
    }
}

}  // namespace rptc

using namespace rptc;

extern "C" int64_t rptc_token_logprobs_workspace_bytes(int64_t rows, int64_t n, int top) {
    (void)rows, (void)n, (void)top;
    return 0;
}

extern "C" int rptc_token_logprobs(const void *logits, int dtype, int64_t ld, const int64_t *targets, float *logprob, float *entropy, float *top_logprobs,
                                   int64_t *top_ids, int64_t rows, int64_t n, int top, void *workspace, int64_t workspace_bytes, rptc_stream_t stream) {
    if (!logits || dtype < 0 || dtype > 2 || (targets && !logprob) || top < 0 || (top > 0 && (!top_logprobs || !top_ids))) return RPTC_ERR_ARG;
    if (rows < 0 || n <= 0 || top > n || ld < n) return RPTC_ERR_SHAPE;
    if (top > 32 || n > (1 << 24) || rows > (1 << 24)) return RPTC_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(logits) & (dtype == 2 ? 3 : 1)) return RPTC_ERR_ALIGN;
    if (int64_t need = rptc_token_logprobs_workspace_bytes(rows, n, top)) {
        if (!workspace || workspace_bytes < need) return RPTC_ERR_ARG;
        if (reinterpret_cast<uintptr_t>(workspace) & 255) return RPTC_ERR_ALIGN;
    }
    if (int e = rptc_check_device()) return e;
    if (rows == 0) return RPTC_OK;
    LogprobParams p = {logits, ld, targets, logprob, entropy, top_logprobs, top_ids, n, top, device_status_word()};
    if (!p.status) return RPTC_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)rows);
    return dtype == 0 ? launch(token_logprobs_kernel<0>, grid, dim3(256), 0, s, p)
           : dtype == 1 ? launch(token_logprobs_kernel<1>, grid, dim3(256), 0, s, p)
                        : launch(token_logprobs_kernel<2>, grid, dim3(256), 0, s, p);
}
