// kv_append.cu -- new K/V rows into the paged cache, rotated to their positions
// on the way, with the rotated queries (velo_cuda_kv_append).
//
// rot(x)_i = x_i cos a - x_{i+D/2} sin a, rot(x)_{i+D/2} = x_i sin a + x_{i+D/2} cos a,
// a = pos * base^(-2i/D).  An angle in f32 loses all its digits far into a long
// context (pos 10^5 leaves 2^-7 of a radian), so the frequency is kept in turns
// as a 64-bit fraction and pos * f wraps modulo one turn by itself.  The sine and
// cosine of the remainder are taken in 64 bits and rounded to f32; both products
// and their sum are rounded to f32 too (no fma), so that a row, and the integers
// an INT8 page truncates it to, have one definition whatever the compiler does.
//
// One block per token: its angles are computed once (a thread per pair) into
// shared memory, then a thread takes 8 rotation pairs of a head, in equal rounds
// when there are more than 256 such items.  A block's time is mostly the latency of
// finding its place (sequence, page, angles) and its rows, so six blocks per SM
// matter more than loads moved up within one (2048 tokens of INT8 pages took 13.5 us with
// them and 11.6 without, before the sine and cosine were taken in 64 bits).
//
// Measured on a B200 against 6552 GB/s: 8533 prompt tokens of 32/32 heads, f32 to f16
// pages, 96 us (1.0); 2048 tokens of 32/8 heads, bf16 to INT8, 12.4 us (0.67, latency);
// 64 single tokens of 64/8 heads 3.3 us.
#include <algorithm>

#include "common/elem.cuh"
#include "common/pdl.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

constexpr int kMaxThreads = 256, kMinBlocks = 6;
constexpr int kErrAppend = 0x6201;

// Number of sequences that start at or before token t, minus one: its sequence
// (the last of several that start at the same token, so empty ones are passed
// over).  A two-level search over blockDim sorted starts each.
__device__ __forceinline__ int find_sequence(const int32_t* start, int B, int t) {
    int lo = 0, n = B;  // the answer lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + (int)blockDim.x - 1) / (int)blockDim.x;
        const int i = (int)threadIdx.x * step;
        const int hit = __syncthreads_count(i < n && start[lo + i] <= t);
        if (hit == 0) return -1;
        lo += (hit - 1) * step;
        n = min(step, n - (hit - 1) * step);
    }
    return lo;
}

// Sequence i's tokens [begin, end): the first block looks at all of them.  Starts that
// do not rise from 0 to n_tokens at most would leave tokens out or move them.
__device__ __forceinline__ void check_start(const KvAppendArgs& a, int i, int begin, int end) {
    if (i < a.B && ((i == 0 && begin != 0) || end < begin || end > a.T)) atomicCAS(a.err, 0, kErrAppend);
}

// This thread's 8 rotation pairs of head `hh` (q heads, then k, then v) of token t.
template <typename In, int D>
__device__ __forceinline__ const In* source(const KvAppendArgs& a, int t, int hh, int i0) {
    const int Hkv = a.kv.n_kv;
    if (hh < a.Hq) return static_cast<const In*>(a.q) + (size_t)t * a.ldq + (size_t)hh * D + i0;
    if (hh < a.Hq + Hkv) return static_cast<const In*>(a.k) + (size_t)t * a.ldk + (size_t)(hh - a.Hq) * D + i0;
    return static_cast<const In*>(a.v) + (size_t)t * a.ldv + (size_t)(hh - a.Hq - Hkv) * D + i0;
}

template <typename In, typename Act, typename Kv, int D>
__global__ void __launch_bounds__(kMaxThreads, kMinBlocks) kv_append_kernel(const __grid_constant__ KvAppendArgs a) {
    constexpr int kLanes = D / 16;  // threads per head, 8 pairs each
    __shared__ float cs[D / 2], sn[D / 2];
    __shared__ int s_seq[3];
    dependent_wait();
    const int t = blockIdx.x;
    const int Hkv = a.kv.n_kv, heads = a.Hq + 2 * Hkv, items = (heads * kLanes + 31) / 32 * 32;
    int b = t, first = t, cached;
    if (!a.seq_start) {
        cached = a.ctx_len[t];
    } else if (a.B <= (int)blockDim.x) {  // a thread per sequence: one round of reads
        const int i = threadIdx.x, total = a.seq_start[a.B];
        const int begin = i < a.B ? a.seq_start[i] : 0, end = i < a.B ? a.seq_start[i + 1] : 0;
        if (t == 0) check_start(a, i, begin, end);
        if (t >= total) return;  // padding rows
        const int len = i < a.B ? a.ctx_len[i] : 0;
        const bool here = i < a.B && begin <= t && t < end;
        if (here) {
            s_seq[0] = i;
            s_seq[1] = begin;
            s_seq[2] = len;
        }
        b = -1;
        if (__syncthreads_or(here)) {
            b = s_seq[0];
            first = s_seq[1];
            cached = s_seq[2];
        }
    } else {
        if (t == 0)
            for (int i = threadIdx.x; i < a.B; i += blockDim.x) check_start(a, i, a.seq_start[i], a.seq_start[i + 1]);
        if (t >= a.seq_start[a.B]) return;
        b = find_sequence(a.seq_start, a.B, t);
        if (b >= 0) {
            first = a.seq_start[b];
            if (t >= a.seq_start[b + 1]) b = -1;
            else cached = a.ctx_len[b];
        }
    }
    if (b < 0) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kErrAppend);
        return;
    }
    const long long pos = (long long)cached + ((long long)t - first);
    const int pi = (int)(pos / kPageTokens), slot = (int)(pos % kPageTokens);
    bool ok = cached >= 0 && pos >= 0 && pos / kPageTokens < a.kv.max_pages;
    uint32_t page = 0;
    if (ok) page = a.kv.page_table[(size_t)b * a.kv.max_pages + pi];
    if (threadIdx.x < D / 2) {
        const uint64_t turn = (uint64_t)pos * a.turns.f[threadIdx.x];
        // a signed fraction of a turn; sincospi takes half turns
        const double half_turns = (double)(int64_t)turn * 1.0842021724855044e-19;  // 2^-63
        double s, c;
        sincospi(half_turns, &s, &c);
        sn[threadIdx.x] = (float)s;
        cs[threadIdx.x] = (float)c;
    }
    ok = ok && page < (uint32_t)a.kv.pool_pages;
    if (!ok && threadIdx.x == 0) atomicCAS(a.err, 0, kErrAppend);
    __syncthreads();
    for (int w = threadIdx.x; w < items; w += blockDim.x) {
        const int hh = w / kLanes, i0 = (w % kLanes) * 8;
        const bool live = hh < heads, is_q = hh < a.Hq, is_v = hh >= a.Hq + Hkv;
        const int h = is_q ? hh : is_v ? hh - a.Hq - Hkv : hh - a.Hq;
        float x0[8], x1[8];
        if (live) {
            const In* src = source<In, D>(a, t, hh, i0);
            load8(src, x0);
            load8(src + D / 2, x1);
            if (!is_v) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = cs[i0 + e], s = sn[i0 + e];
                    const float y0 = __fsub_rn(__fmul_rn(x0[e], c), __fmul_rn(x1[e], s));
                    const float y1 = __fadd_rn(__fmul_rn(x0[e], s), __fmul_rn(x1[e], c));
                    x0[e] = y0;
                    x1[e] = y1;
                }
            }
            if (is_q) {
                Act* dst = static_cast<Act*>(a.q_out) + ((size_t)t * a.Hq + h) * D;
                store8(dst + i0, x0);
                store8(dst + i0 + D / 2, x1);
            }
        }
        const size_t row = ((size_t)page * Hkv + h) * kPageTokens + slot;
        void* pool = is_v ? a.kv.v_pool : a.kv.k_pool;
        if constexpr (sizeof(Kv) == 1) {  // quantise: the head's lanes share the maximum
            float mx = 0.0f;
            if (live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fmaxf(fabsf(x0[e]), fabsf(x1[e])));
            }
#pragma unroll
            for (int o = kLanes / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (!live || is_q) continue;
            float inv = mx > 0.0f ? __fdiv_rn(127.0f, mx) : 0.0f;
            if (inv == INFINITY) inv = 0.0f;  // a row below 2^-121: its scale is 0 as well
            const __half scale = __float2half_rn(__fdiv_rn(mx, 127.0f));
            uint32_t w0[2] = {0, 0}, w1[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int q0 = (int)__fmul_rn(x0[e], inv), q1 = (int)__fmul_rn(x1[e], inv);  // truncation
                w0[e / 4] |= (uint32_t)(q0 & 0xff) << (8 * (e % 4));
                w1[e / 4] |= (uint32_t)(q1 & 0xff) << (8 * (e % 4));
                x0[e] = (float)q0 * __half2float(scale);
                x1[e] = (float)q1 * __half2float(scale);
            }
            if (ok) {
                int8_t* dst = static_cast<int8_t*>(pool) + row * D;
                *reinterpret_cast<uint2*>(dst + i0) = make_uint2(w0[0], w0[1]);
                *reinterpret_cast<uint2*>(dst + i0 + D / 2) = make_uint2(w1[0], w1[1]);
                if (i0 == 0) (is_v ? a.kv.v_scale : a.kv.k_scale)[row] = scale;
            }
        } else {
            if (!live || is_q) continue;
            if (ok) {
                Kv* dst = static_cast<Kv*>(pool) + row * D;
                store8(dst + i0, x0);
                store8(dst + i0 + D / 2, x1);
            }
        }
        if (a.k_out) {
            Act* dst = static_cast<Act*>(is_v ? a.v_out : a.k_out) + ((size_t)t * Hkv + h) * D;
            store8(dst + i0, x0);
            store8(dst + i0 + D / 2, x1);
        }
    }
}

template <typename In, typename Act, typename Kv>
cudaError_t launch_typed(const KvAppendArgs& a, cudaStream_t s) {
    // equal rounds of at most 256 threads (and one per rotation pair, for the angles)
    const int items = (a.Hq + 2 * a.kv.n_kv) * (a.kv.head_dim / 16), rounds = (items + kMaxThreads - 1) / kMaxThreads;
    const int threads = std::max((items + rounds - 1) / rounds + 31 & ~31, 64);
    return launch_dependent(a.kv.head_dim == 64 ? kv_append_kernel<In, Act, Kv, 64> : kv_append_kernel<In, Act, Kv, 128>,
                            dim3(a.T), threads, 0, 1, s, a);
}

template <typename In>
cudaError_t launch_from(const KvAppendArgs& a, cudaStream_t s) {
    if (a.kv.kv_dtype == VELO_KV_F32) return launch_typed<In, float, float>(a, s);
    if (a.kv.kv_dtype == VELO_KV_INT8) return launch_typed<In, __half, int8_t>(a, s);
    return launch_typed<In, __half, __half>(a, s);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
    if (a.in_dtype == VELO_ELEM_F32) return launch_from<float>(a, s);
    if (a.in_dtype == VELO_ELEM_F16) return launch_from<__half>(a, s);
    return launch_from<__nv_bfloat16>(a, s);
}

}  // namespace velo
