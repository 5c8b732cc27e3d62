// token_logprobs.cu -- log probability of given tokens, entropy and the best
// alternatives of each logits row (velo_cuda_token_logprobs).
//
// With d = x / T - m, m the row's maximum of x / T: Z = sum e^d,
// logprob = d[token] - log Z, entropy = log Z - sum d e^d / Z.  Top n: the rows's
// (value, lowest index) order as whole numbers, the n-th largest value found by
// a radix select over 8-bit digits, equal values taken in index order.
//
// One block per row, one pass for the maximum and one for the sums.
#include "common/elem.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kErrToken = 0x6221;

// Value order as unsigned whole numbers: -0 equals 0, NaN below -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
__device__ __forceinline__ float row_at(const T* row, int i) {
    return to_f32(row[i]);
}

__device__ __forceinline__ float nan_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The n largest (value, lowest index) of the row, any values: ids[0..n) in
// descending order.  hist: 256 counters, all threads call it.
template <typename T>
__device__ void radix_top(const T* row, int V, int n, uint32_t* hist, uint32_t* keys, uint32_t* ids, uint32_t* out) {
    __shared__ uint32_t s_prefix, s_left, s_count;
    __shared__ uint32_t warp_cnt[kWarps];
    if (threadIdx.x == 0) {
        s_prefix = 0;
        s_left = (uint32_t)n;  // how many of the elements that share the prefix belong to the top
        s_count = 0;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = threadIdx.x; i < V; i += kThreads) {
            const uint32_t k = order_key(row_at(row, i));
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t left = s_left;
            int d = 255;
            while (hist[d] < left) left -= hist[d--];
            s_left = left;
            s_prefix = prefix | ((uint32_t)d << shift);
        }
        __syncthreads();
    }
    // s_prefix is the n-th largest key; s_left of its holders, in index order, belong to the top
    const uint32_t kth = s_prefix, ties = s_left;
    uint32_t seen = 0;
    for (int base = 0; base < V; base += kThreads) {
        const int i = base + threadIdx.x;
        const uint32_t k = i < V ? order_key(row_at(row, i)) : 0u;
        const bool tie = i < V && k == kth;
        const uint32_t bal = __ballot_sync(0xffffffffu, tie);
        const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) warp_cnt[w] = __popc(bal);
        __syncthreads();
        uint32_t before = seen + __popc(bal & ((1u << lane) - 1));
        for (int j = 0; j < kWarps; ++j) {
            if (j < w) before += warp_cnt[j];
            seen += warp_cnt[j];
        }
        if (i < V && (k > kth || (tie && before < ties))) {
            const uint32_t at = atomicAdd(&s_count, 1u);
            keys[at] = k;
            ids[at] = (uint32_t)i;
        }
        __syncthreads();
    }
    if ((int)threadIdx.x < n) {
        const uint32_t k = keys[threadIdx.x], id = ids[threadIdx.x];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += keys[j] > k || (keys[j] == k && ids[j] < id);
        out[rank] = id;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const TokenLogprobsArgs a) {
    __shared__ float red[kWarps], red2[kWarps];
    __shared__ uint32_t hist[256], keys[kMaxTop], ids[kMaxTop], best[kMaxTop];
    const int r = blockIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const T* row = static_cast<const T*>(a.logits) + (size_t)r * a.ldl;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.V; i += kThreads) m = nan_max(m, row_at(row, i));
    for (int o = 16; o; o >>= 1) m = nan_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[w] = m;
    __syncthreads();
    m = red[0];
    for (int i = 1; i < kWarps; ++i) m = nan_max(m, red[i]);
    __syncthreads();
    const float mt = m == -INFINITY ? 0.0f : m * a.inv_t;
    float z = 0.0f, y = 0.0f;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
        const float d = fmaf(row_at(row, i), a.inv_t, -mt), e = expf(d);
        z += e;
        if (e != 0.0f) y += e * d;
    }
    for (int o = 16; o; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    if (lane == 0) {
        red[w] = z;
        red2[w] = y;
    }
    __syncthreads();
    z = y = 0.0f;
    for (int i = 0; i < kWarps; ++i) {
        z += red[i];
        y += red2[i];
    }
    const float log_z = logf(z);
    auto lp_of = [&](uint32_t i) {
        const float d = fmaf(row_at(row, (int)i), a.inv_t, -mt);
        return d == -INFINITY ? (log_z == log_z ? d : log_z) : d - log_z;
    };
    if (threadIdx.x == 0) {
        if (a.logprob) {
            const uint32_t t = a.tokens[r];
            if (t >= (uint32_t)a.V) atomicCAS(a.err, 0, kErrToken);
            a.logprob[r] = t < (uint32_t)a.V ? lp_of(t) : __int_as_float(0x7fc00000);
        }
        if (a.entropy) a.entropy[r] = m == -INFINITY ? 0.0f : log_z - y / z;
    }
    if (a.n_top > 0) {
        radix_top(row, a.V, a.n_top, hist, keys, ids, best);
        for (int i = threadIdx.x; i < a.n_top; i += kThreads) {
            a.top_tokens[(size_t)r * a.n_top + i] = best[i];
            a.top_logprobs[(size_t)r * a.n_top + i] = lp_of(best[i]);
        }
    }
}

}  // namespace

cudaError_t launch_token_logprobs(const TokenLogprobsArgs& a, int, cudaStream_t s) {
    if (a.dtype == VELO_ELEM_F32)
        logprobs_kernel<float><<<a.M, kThreads, 0, s>>>(a);
    else if (a.dtype == VELO_ELEM_F16)
        logprobs_kernel<__half><<<a.M, kThreads, 0, s>>>(a);
    else
        logprobs_kernel<__nv_bfloat16><<<a.M, kThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace velo
