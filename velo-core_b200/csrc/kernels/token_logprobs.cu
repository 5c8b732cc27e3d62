// token_logprobs.cu -- log probability of given tokens, entropy and the best
// alternatives of each logits row (velo_cuda_token_logprobs).
//
// With m the row's maximum, k = log2(e) / T, u = (x - m) k: Z = sum 2^u, Y = sum u 2^u,
// log probability = (x[token] - m) / T - ln Z, entropy = ln Z - ln 2 Y / Z.
// Each logit is read once from HBM, which bounds the kernel.
//
// A block (or, with few rows, a cluster of up to 8 blocks) streams a row through
// 16 KB stages filled by cp.async; every thread copies the vectors it consumes
// itself, so the stream needs no barrier.  A thread keeps its own (m, Z, Y)
// and, per sixteenth of the row, the maximum of what it saw.
//
// The n best: the ceil(n / 8)-th largest thread maximum of every warp, least of
// them over the warps, is a bound that at least n elements reach; only the
// (thread, sixteenth) pieces whose maximum reaches it are read again (from L2) and
// their elements at or above it listed -- a few dozen in an ordinary row.  Should
// the list overflow (ties, ordered rows), it is rebuilt with a higher bound and
// the ties of the bound are taken in index order.  Positions in the list order
// decide the rank, so the result does not depend on the order of arrival.
//
// With a cluster each block sends its sums and its own n best to the first one's
// shared memory, which ranks them.
#include <algorithm>

#include "common/elem.cuh"
#include "common/sm100.cuh"
#include "common/smem_attr.cuh"
#include "common/spec_math.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

using sm100::ex2_approx;
using sm100::smem_u32;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kErrToken = 0x6221;
constexpr int kVecs = 4;                              // 16-byte vectors per thread and tile
constexpr int kTileVecs = kVecs * kThreads;           // 16 KB
constexpr int kStages = 3;
constexpr int kSlots = 16;                            // pieces of the row with their own maxima
constexpr int kList = 512;                            // candidates before the bound is raised
constexpr int kMaxCluster = 8;
constexpr float kLn2 = 0.693147180559945309f;

// Dynamic shared memory.  After the stream the ring holds the selection's lists.
constexpr int kRingBytes = kStages * kTileVecs * 16;
constexpr int kSlotOfs = kRingBytes;
constexpr int kInboxOfs = kSlotOfs + kSlots * kThreads * 4;
constexpr int kInboxStride = kMaxTop * 8 + 16;        // sorted keys, then m, Z, Y, count
constexpr int kSmemOne = kInboxOfs + kInboxStride;
constexpr int kSmemCluster = kInboxOfs + kMaxCluster * kInboxStride;
constexpr int kWorkOfs = (kList + kMaxTop) * 8;       // u16 pieces to read again
static_assert(kWorkOfs + kSlots * kThreads * 2 <= kRingBytes, "lists fit the ring");
static_assert(kMaxCluster * kMaxTop <= kList + kMaxTop, "a cluster's lists fit the list");

// Value order as unsigned whole numbers: -0 equals 0, NaN below -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == 0u) return __int_as_float(0x7fc00000);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// (value, lowest index) order as one number
__device__ __forceinline__ unsigned long long full_key(uint32_t k, int i) {
    return (unsigned long long)k << 32 | (uint32_t)~i;
}

__device__ __forceinline__ float nan_max(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const float*, uint4 v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const __half*, uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const __nv_bfloat16*, uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Running sums: m is the largest logit, Z and Y belong to u = (x - m) k.  (x - m
// rather than one fma: a row masked with the type's lowest value must not overflow.)
struct Sums {
    float m, z, y;
};
// What x is measured from while the largest logit is m.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Sums join(Sums a, Sums b, float k) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    // u' = u + d, d = (own m - new m) k; a part without finite elements has Z = Y = 0
    const float da = a.m == -INFINITY ? 0.0f : (a.m - r.m) * k;
    const float db = b.m == -INFINITY ? 0.0f : (b.m - r.m) * k;
    const float fa = ex2_approx(da), fb = ex2_approx(db);
    r.z = a.z * fa + b.z * fb;
    // (a factor of 0 must not meet an infinite difference)
    r.y = fa * a.y + fb * b.y + (fa > 0.0f ? fa * da * a.z : 0.0f) + (fb > 0.0f ? fb * db * b.z : 0.0f);
    return r;
}
__device__ __forceinline__ void raise(Sums& s, float m, float k) {
    if (m > s.m) s = join(s, Sums{m, 0.0f, 0.0f}, k);
}
// Adds 2^u and u 2^u of two logits to (z, y); -inf adds 0, not 0 * inf, NaN stays.
__device__ __forceinline__ void add_two(float2& z, float2& y, float x0, float x1, float2 minus_m, float2 k) {
    float2 u = __fmul2_rn(__fadd2_rn(make_float2(x0, x1), minus_m), k);
    u.x = nan_max(u.x, -200.0f);
    u.y = nan_max(u.y, -200.0f);
    const float2 e = make_float2(ex2_approx(u.x), ex2_approx(u.y));
    z = __fadd2_rn(z, e);
    y = __ffma2_rn(e, u, y);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_first(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void store_remote(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Rank of every key of list[0 .. c), c <= blockDim * 3 (all distinct): calls
// put(rank, key).
template <typename F>
__device__ __forceinline__ void rank_list(const unsigned long long* list, int c, F put) {
    for (int i = threadIdx.x; i < c; i += kThreads) {
        const unsigned long long k = list[i];
        int r = 0;
        for (int j = 0; j < c; ++j) r += list[j] > k;
        put(r, k);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_kernel(const TokenLogprobsArgs a, int cluster) {
    constexpr int kN = Vec<T>::n;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums s_part[kWarps];
    __shared__ uint32_t s_bound[kWarps];
    __shared__ int s_count, s_work, s_warp[kWarps];
    __shared__ unsigned long long s_raise;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / cluster, part = blockIdx.x % cluster;
    if (cluster > 1) cluster_arrive();  // the first block's inbox may be written once all have started
    const T* row = static_cast<const T*>(a.logits) + (size_t)r * a.ldl;
    const float k = a.inv_t * kLog2e;
    float tok_x = 0.0f;
    uint32_t tok = 0;
    if (a.logprob && part == 0 && tid == 0) {
        tok = a.tokens[r];
        if (tok < (uint32_t)a.V) tok_x = to_f32(row[tok]);
    }

    // elements [lo, hi) of this block: aligned vectors, and the row's ragged ends
    const int head = min(a.V, (int)((16 - (uintptr_t)row % 16) % 16 / sizeof(T)));
    const int nv_row = (a.V - head) / kN;
    const int v0 = (int)((long long)nv_row * part / cluster), v1 = (int)((long long)nv_row * (part + 1) / cluster);
    const int lo = part == 0 ? 0 : head + v0 * kN, hi = part == cluster - 1 ? a.V : head + v1 * kN;
    const int nv = v1 - v0, tiles = (nv + kTileVecs - 1) / kTileVecs, per_slot = (tiles + kSlots - 1) / kSlots;
    const T* body = row + head + (size_t)v0 * kN;
    float* slot_max = reinterpret_cast<float*>(smem + kSlotOfs);

    auto issue = [&](int tile) {
        if (tile < tiles) {
            const uint32_t st = smem_u32(smem) + (tile % kStages) * kTileVecs * 16 + tid * 16;
#pragma unroll
            for (int q = 0; q < kVecs; ++q) {
                const int v = tile * kTileVecs + q * kThreads + tid;
                const int n = v < nv ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(st + q * kThreads * 16),
                             "l"(body + (size_t)(n ? v : 0) * kN), "r"(n)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kStages; ++i) issue(i);

    Sums s{-INFINITY, 0.0f, 0.0f};
    // the ragged ends, one element per thread: index, or -1
    int ragged = -1;
    if (tid < head && part == 0) ragged = tid;
    const int tail0 = head + nv_row * kN;
    if (part == cluster - 1 && tid >= 32 && tid - 32 < a.V - tail0) ragged = tail0 + tid - 32;
    if (ragged >= 0) {
        const float x = to_f32(row[ragged]);
        raise(s, x, k);
        float2 z = f2(0.0f), y = f2(0.0f);
        add_two(z, y, x, -INFINITY, f2(-base_of(s.m)), f2(k));
        s.z += z.x;
        s.y += y.x;
    }

    float piece = -INFINITY;
    for (int tile = 0; tile < tiles; ++tile) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        const uint8_t* st = smem + (tile % kStages) * kTileVecs * 16 + tid * 16;
        const bool full = (tile + 1) * kTileVecs <= nv;
        float x[kVecs * kN];
#pragma unroll
        for (int q = 0; q < kVecs; ++q) unpack(row, *reinterpret_cast<const uint4*>(st + q * kThreads * 16), x + q * kN);
        if (!full) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
                if (tile * kTileVecs + q * kThreads + tid >= nv) {
#pragma unroll
                    for (int e = 0; e < kN; ++e) x[q * kN + e] = -INFINITY;
                }
        }
        issue(tile + kStages);  // the stage's values are in registers
        float m = x[0];
#pragma unroll
        for (int i = 1; i < kVecs * kN; ++i) m = fmaxf(m, x[i]);
        piece = fmaxf(piece, m);
        raise(s, m, k);
        const float2 minus_m = f2(-base_of(s.m));
        float2 z = f2(0.0f), y = f2(0.0f);
#pragma unroll
        for (int i = 0; i < kVecs * kN; i += 2) add_two(z, y, x[i], x[i + 1], minus_m, f2(k));
        s.z += z.x + z.y;
        s.y += y.x + y.y;
        if ((tile + 1) % per_slot == 0 || tile + 1 == tiles) {
            slot_max[tile / per_slot * kThreads + tid] = piece;
            piece = -INFINITY;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the block's sums, and each warp's bound for the selection
    const uint32_t top_key = order_key(s.m);
    Sums w = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Sums x{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.z, o),
                     __shfl_xor_sync(0xffffffffu, w.y, o)};
        // the same order on both sides of the exchange
        w = lane & o ? join(x, w, k) : join(w, x, k);
    }
    const int full_warps = min(kWarps, nv / 32);  // warps whose every lane has data
    const int each = full_warps ? (a.n_top + full_warps - 1) / full_warps : 0;
    if (a.n_top) {
        uint32_t key = top_key, bound = 0;
        for (int i = 0; i < each; ++i) {
            bound = __reduce_max_sync(0xffffffffu, key);
            const uint32_t who = __ballot_sync(0xffffffffu, key == bound);
            if (lane == __ffs(who) - 1) key = 0;
        }
        if (lane == 0) s_bound[warp] = bound;
    }
    if (lane == 0) s_part[warp] = w;
    __syncthreads();
    s = s_part[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) s = join(s, s_part[i], k);

    // ---- the block's n best, sorted, into its inbox
    unsigned long long* list = reinterpret_cast<unsigned long long*>(smem);
    uint16_t* work = reinterpret_cast<uint16_t*>(smem + kWorkOfs);
    unsigned long long* mine = reinterpret_cast<unsigned long long*>(smem + kInboxOfs);
    const int want = min(a.n_top, hi - lo);
    if (a.n_top) {
        // every element with key > bound (or >= if ties) into the list; the number found
        auto collect = [&](uint32_t bound, bool ties) {
            __syncthreads();
            if (tid == 0) s_count = s_work = 0;
            __syncthreads();
            for (int i = 0; i * per_slot < tiles; ++i) {
                const uint32_t mk = order_key(slot_max[i * kThreads + tid]);
                if (mk > bound || (ties && mk == bound)) work[atomicAdd(&s_work, 1)] = (uint16_t)(i * kThreads + tid);
            }
            auto offer = [&](float x, int i) {
                const uint32_t kx = order_key(x);
                if (kx > bound || (ties && kx == bound)) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < kList) list[at] = full_key(kx, i);
                }
            };
            if (ragged >= 0) offer(to_f32(row[ragged]), ragged);
            __syncthreads();
            const int per = per_slot * kVecs, n = s_work * per;
            for (int i = tid; i < n; i += kThreads) {
                const int p = work[i / per], j = i % per;
                const int v = ((p / kThreads) * per_slot + j / kVecs) * kTileVecs + (j % kVecs) * kThreads + p % kThreads;
                if (v >= nv || (p / kThreads) * per_slot + j / kVecs >= tiles) continue;
                float x[kN];
                unpack(row, __ldg(reinterpret_cast<const uint4*>(body + (size_t)v * kN)), x);
#pragma unroll
                for (int e = 0; e < kN; ++e) offer(x[e], head + (v0 + v) * kN + e);
            }
            __syncthreads();
            return s_count;
        };
        // appends the first `need` elements equal to the bound, in index order
        auto add_ties = [&](uint32_t bound, int c, int need) {
            int seen = 0;
            for (int base = lo; base < hi && seen < need; base += kThreads) {
                const int i = base + tid;
                const bool tie = i < hi && order_key(to_f32(row[i])) == bound;
                const uint32_t bal = __ballot_sync(0xffffffffu, tie);
                if (lane == 0) s_warp[warp] = __popc(bal);
                __syncthreads();
                int before = seen + __popc(bal & ((1u << lane) - 1));
#pragma unroll
                for (int j = 0; j < kWarps; ++j) {
                    if (j < warp) before += s_warp[j];
                    seen += s_warp[j];
                }
                if (tie && before < need) list[c + before] = full_key(bound, i);
                __syncthreads();
            }
            return c + min(seen, need);
        };
        uint32_t bound = full_warps ? 0xffffffffu : 0u;
        for (int i = 0; i < full_warps; ++i) bound = min(bound, s_bound[i]);
        int c = collect(bound, true);
        if (c > kList) {
            while ((c = collect(bound, false)) > kList) {
                // a higher bound: the want-th best of those listed
                rank_list(list, kList, [&](int rank, unsigned long long key) {
                    if (rank == want - 1) s_raise = key;
                });
                __syncthreads();
                bound = (uint32_t)(s_raise >> 32);
            }
            if (c < want) c = add_ties(bound, c, want - c);
        } else if (c < want) {  // NaN entries among the best: below everything else, in index order
            c = collect(0u, false);
            if (c < want) c = add_ties(0u, c, want - c);
        }
        __syncthreads();
        rank_list(list, c, [&](int rank, unsigned long long key) {
            if (rank < want) mine[rank] = key;
        });
        __syncthreads();
    }

    // ---- over the cluster
    if (cluster > 1) {
        cluster_wait();  // all blocks have started
        if (part != 0) {
            const uint32_t box = map_to_first(smem_u32(smem + kInboxOfs + part * kInboxStride));
            for (int i = tid; i < want; i += kThreads) store_remote(box + i * 8, mine[i]);
            if (tid == 0) {
                store_remote(box + kMaxTop * 8,
                             (unsigned long long)__float_as_uint(s.z) << 32 | __float_as_uint(s.m));
                store_remote(box + kMaxTop * 8 + 8, (unsigned long long)(uint32_t)want << 32 | __float_as_uint(s.y));
            }
        }
        cluster_arrive();  // release
        cluster_wait();    // acquire (the others only stay until the first has their data)
        if (part != 0) return;
        int c = want;
        for (int i = tid; i < want; i += kThreads) list[i] = mine[i];
        for (int p = 1; p < cluster; ++p) {
            const uint8_t* box = smem + kInboxOfs + p * kInboxStride;
            const float* f = reinterpret_cast<const float*>(box + kMaxTop * 8);
            s = join(s, Sums{f[0], f[1], f[2]}, k);
            const int n = __float_as_int(f[3]);
            for (int i = tid; i < n; i += kThreads) list[c + i] = reinterpret_cast<const unsigned long long*>(box)[i];
            c += n;
        }
        __syncthreads();
        rank_list(list, c, [&](int rank, unsigned long long key) {
            if (rank < a.n_top) mine[rank] = key;
        });
        __syncthreads();
    }

    // NaN and +inf have made Z NaN; Z is 0 only for a row of -inf
    const float log_z = logf(s.z);
    auto lp = [&](float x) {
        if (log_z != log_z) return log_z;
        const float d = x - base_of(s.m);
        return d == -INFINITY ? d : fmaf(d, a.inv_t, -log_z);
    };
    if (tid == 0) {
        if (a.logprob) {
            if (tok >= (uint32_t)a.V) atomicCAS(a.err, 0, kErrToken);
            a.logprob[r] = tok < (uint32_t)a.V ? lp(tok_x) : __int_as_float(0x7fc00000);
        }
        if (a.entropy) a.entropy[r] = s.z == 0.0f ? 0.0f : log_z - kLn2 * (s.y / s.z);
    }
    for (int i = tid; i < a.n_top; i += kThreads) {
        const unsigned long long key = mine[i];
        a.top_tokens[(size_t)r * a.n_top + i] = ~(uint32_t)key;
        a.top_logprobs[(size_t)r * a.n_top + i] = lp(key_value((uint32_t)(key >> 32)));
    }
}

// Blocks per row: enough for two blocks per SM, as long as each keeps a tile's worth.
int cluster_of(const TokenLogprobsArgs& a, int sm_count) {
    const int per_tile = kTileVecs * (a.dtype == VELO_ELEM_F32 ? 4 : 8);
    int c = 1;
    while (c < kMaxCluster && (long long)a.M * c < 2LL * sm_count && a.V / (2 * c) >= per_tile) c *= 2;
    return c;
}

template <typename T>
cudaError_t launch_typed(const TokenLogprobsArgs& a, int sm_count, cudaStream_t s) {
    static SmemAttr attr;
    const int cluster = cluster_of(a, sm_count);
    const int smem = cluster > 1 ? kSmemCluster : kSmemOne;
    cudaError_t e = ensure_smem(attr, token_logprobs_kernel<T>, kSmemCluster);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = (unsigned)a.M * cluster;
    cfg.blockDim = kThreads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a, cluster);
}

}  // namespace

cudaError_t launch_token_logprobs(const TokenLogprobsArgs& a, int sm_count, cudaStream_t s) {
    if (a.dtype == VELO_ELEM_F32) return launch_typed<float>(a, sm_count, s);
    if (a.dtype == VELO_ELEM_F16) return launch_typed<__half>(a, sm_count, s);
    return launch_typed<__nv_bfloat16>(a, sm_count, s);
}

}  // namespace velo
