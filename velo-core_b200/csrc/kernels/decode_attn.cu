// decode_attn.cu -- attention of one query token per sequence over the paged
// cache (velo_cuda_decode_attention).
//
// One block of four warps per (sequence, head): warp w takes tokens w, w + 4,
// ...; a lane holds D / 32 dimensions of q and of the running output; online
// softmax per warp, the four states merged through shared memory.
#include "common/elem.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

constexpr int kErrSeqLen = 0x6211, kErrPage = 0x6212;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

template <typename Act, typename Kv, int D>
__global__ void __launch_bounds__(128) decode_attn_kernel(const DecodeAttnArgs a) {
    constexpr int R = D / 32;
    __shared__ float sm[4], sl[4], so[4][D];
    const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq;
    const int Hkv = a.kv.n_kv, hk = h / (a.Hq / Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int len = a.seq_len[b];
    if (len < 0 || len > a.kv.max_pages * kPageTokens) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrSeqLen);
        len = len < 0 ? 0 : a.kv.max_pages * kPageTokens;
    }
    float q[R], o[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r)
        q[r] = to_f32(static_cast<const Act*>(a.q)[(size_t)b * a.ldq + (size_t)h * D + r * 32 + lane]) * a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f;
    for (int t = warp; t < len; t += 4) {
        const uint32_t pg = a.kv.page_table[(size_t)b * a.kv.max_pages + t / kPageTokens];
        if (pg >= (uint32_t)a.kv.pool_pages) {
            if (lane == 0) atomicCAS(a.err, 0, kErrPage);
            continue;
        }
        const size_t row = ((size_t)pg * Hkv + hk) * kPageTokens + t % kPageTokens;
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) s += q[r] * to_f32(static_cast<const Kv*>(a.kv.k_pool)[row * D + r * 32 + lane]);
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        float vs = 1.0f;
        if constexpr (sizeof(Kv) == 1) {
            s *= __half2float(a.kv.k_scale[row]);
            vs = __half2float(a.kv.v_scale[row]);
        }
        const float mn = fmaxf(m, s), alpha = exp2f(m - mn), p = exp2f(s - mn);
        m = mn;
        l = l * alpha + p;
#pragma unroll
        for (int r = 0; r < R; ++r)
            o[r] = o[r] * alpha + p * vs * to_f32(static_cast<const Kv*>(a.kv.v_pool)[row * D + r * 32 + lane]);
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) so[warp][r * 32 + lane] = o[r];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w]);
    for (int w = 0; w < 4; ++w) L += M == -INFINITY ? 0.0f : sl[w] * exp2f(sm[w] - M);
    for (int d = threadIdx.x; d < D; d += 128) {
        float x = 0.0f;
        if (M != -INFINITY)
            for (int w = 0; w < 4; ++w) x += so[w][d] * exp2f(sm[w] - M);
        static_cast<Act*>(a.out)[((size_t)b * a.Hq + h) * D + d] = (Act)(L > 0.0f ? x / L : 0.0f);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[(size_t)b * a.Hq + h] = L > 0.0f ? (M + log2f(L)) * kLn2 : -INFINITY;
}

template <typename Act, typename Kv>
cudaError_t launch_typed(const DecodeAttnArgs& a, cudaStream_t s) {
    if (a.kv.head_dim == 64)
        decode_attn_kernel<Act, Kv, 64><<<a.B * a.Hq, 128, 0, s>>>(a);
    else
        decode_attn_kernel<Act, Kv, 128><<<a.B * a.Hq, 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t decode_attn_workspace(int, int, int, int) { return 16; }

cudaError_t launch_decode_attention(const DecodeAttnArgs& a, int, cudaStream_t s) {
    if (a.kv.kv_dtype == VELO_KV_F32) return launch_typed<float, float>(a, s);
    if (a.kv.kv_dtype == VELO_KV_INT8) return launch_typed<__half, int8_t>(a, s);
    return launch_typed<__half, __half>(a, s);
}

}  // namespace velo
