// token_logprobs.cu -- log probability of given tokens, entropy and the best
// alternatives of each logits row (velo_cuda_token_logprobs).
//
// With m the row's maximum so far, k = log2(e) / T, u = (x - m) k: Z = sum 2^u, Y = sum u 2^u,
// log probability = (x[token] - m) / T - ln Z, entropy = ln Z - ln 2 Y / Z.
// Each logit is read once from HBM, which bounds the kernel.
//
// A block (or, with few rows, a cluster of up to 8 blocks) streams a row through
// 16 KB stages filled by cp.async; every thread copies the vectors it consumes
// itself, so the stream needs no barrier.  A thread keeps its own (m, Z, Y)
// and, per sixteenth of the row, the maximum of what it saw.
//
// The n best: the n-th largest of some of the threads' maxima is a bound that at
// least n elements reach; only the (thread, sixteenth) pieces whose maximum
// reaches it are read again and their elements at or above it listed -- little
// more than n in an ordinary row.  Should
// the list overflow (ties, ordered rows), it is rebuilt with a higher bound and
// the ties of the bound are taken in index order.  Positions in the list order
// decide the rank, so the result does not depend on the order of arrival.
//
// With a cluster each block sends its sums and its own n best to the first one's
// shared memory, which ranks them.
//
// Measured on a B200 against 6552 GB/s: 2048 rows of 128256 f32, 20 best, 184 us back
// to back (0.87; the stream alone 170, the rest are selections that no other block of
// the SM hides); 576 rows of 32000 bf16, 8 best, 13.6 us on the device, 14.4 as eager calls
// (one wave of blocks: launch, stream and selection in a row); one row of 128256 f32 7.9 us
// (latency), 64 rows 11.5.
#include <algorithm>
#include <type_traits>

#include "common/elem.cuh"
#include "common/pdl.cuh"
#include "common/sm100.cuh"
#include "common/smem_attr.cuh"
#include "common/spec_math.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

using sm100::ex2_approx;
using sm100::smem_u32;

constexpr int kErrToken = 0x6221;
constexpr int kVecs = 4;                              // 16-byte vectors per thread and tile
constexpr int kSlots = 16;                            // pieces of the row with their own maxima
constexpr int kList = 512;                            // candidates before the bound is raised
constexpr int kMaxCluster = 8;
constexpr size_t kShortRow = 16384;                   // bytes of a row that 64 threads take
constexpr float kLn2 = 0.693147180559945309f;

constexpr int kInboxStride = kMaxTop * 8 + 16;  // sorted keys, then m, Z, Y, count

// A block of kThreads and its dynamic shared memory: the ring (after the stream: the
// candidates and the pieces to read again), the pieces' maxima, the inbox.
// Two stages let four blocks share an SM.
template <int kThreads, int kStages>
struct Block {
    static constexpr int kWarps = kThreads / 32;
    static constexpr int kPerSm = kThreads == 64 ? 16 : kStages == 2 ? 4 : 2;
    static constexpr int kTileVecs = kVecs * kThreads;  // 16 KB with 256 threads
    static constexpr int kRingBytes = kStages * kTileVecs * 16;
    static constexpr int kWorkOfs = (kList + kMaxTop) * 8;
    static constexpr int kSlotOfs = kRingBytes;
    static constexpr int kSmemOne = kSlotOfs + kSlots * kThreads * 4;
    static constexpr int kInboxOfs = kSmemOne;
    static constexpr int kSmemCluster = kInboxOfs + kMaxCluster * kInboxStride;
    static_assert(kWorkOfs + kSlots * kThreads * 2 <= kRingBytes, "lists fit the ring");
};
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
// What x is measured from.
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
// Sums over the first `lanes` lanes of a warp (a power of two), in lane 0.
__device__ __forceinline__ Sums warp_join(Sums s, float k, int lanes) {
    float m = s.m;
    for (int o = lanes / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    s = join(s, Sums{m, 0.0f, 0.0f}, k);
    for (int o = lanes / 2; o; o >>= 1) {
        s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    return s;
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

// The .aligned forms take a warp's threads together, which branches on the thread before them
// do not promise by themselves.
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_to_first(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void store_remote(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Rank of every key of list[0 .. c) (all distinct): calls put(rank, key).
template <int kThreads, typename F>
__device__ __forceinline__ void rank_list(const unsigned long long* list, int c, F put) {
    for (int i = threadIdx.x; i < c; i += kThreads) {
        const unsigned long long k = list[i];
        int r = 0;
        for (int j = 0; j < c; ++j) r += list[j] > k;
        put(r, k);
    }
}

// This block's part of a row: elements [lo, hi), of them nv whole 16-byte vectors
// from `body` on (element `first`); the row's ragged ends belong to its first
// and last part.
template <typename T>
struct Part {
    const T* row;
    const T* body;
    int first, nv, lo, hi;
};

template <typename T, int kThreads, int kStages>
__global__ void __launch_bounds__(kThreads, Block<kThreads, kStages>::kPerSm) token_logprobs_kernel(
    const TokenLogprobsArgs a, int log_cluster) {
    using S = Block<kThreads, kStages>;
    constexpr int kN = Vec<T>::n, kWarps = S::kWarps, kTileVecs = S::kTileVecs;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums s_part[kWarps];
    __shared__ __align__(16) uint32_t s_bound[kWarps * 32 + 4];
    __shared__ int s_count, s_work, s_warp[kWarps];
    __shared__ unsigned long long s_raise;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cluster = 1 << log_cluster, part = blockIdx.x & (cluster - 1), r = blockIdx.x >> log_cluster;
    dependent_wait();
    if (cluster > 1) cluster_arrive();  // the first block's inbox may be written once all have started
    const float k = a.inv_t * kLog2e;
    float* slot_max = reinterpret_cast<float*>(smem + S::kSlotOfs);
    unsigned long long* list = reinterpret_cast<unsigned long long*>(smem);
    uint16_t* work = reinterpret_cast<uint16_t*>(smem + S::kWorkOfs);

    Part<T> p;
    {
        p.row = static_cast<const T*>(a.logits) + (size_t)r * a.ldl;
        const int head = min(a.V, (int)((16 - (uintptr_t)p.row % 16) % 16 / sizeof(T)));
        const int nv_row = (a.V - head) / kN;  // < 2^22
        const int v0 = (nv_row * part) >> log_cluster, v1 = (nv_row * (part + 1)) >> log_cluster;
        p.first = head + v0 * kN;
        p.nv = v1 - v0;
        p.lo = part == 0 ? 0 : p.first;
        p.hi = part == cluster - 1 ? a.V : head + v1 * kN;
        p.body = p.row + p.first;
    }
    const int nv = p.nv, whole_tiles = nv / kTileVecs, tiles = (nv + kTileVecs - 1) / kTileVecs;
    const int per_slot = (tiles + kSlots - 1) / kSlots;
    const uint32_t ring = smem_u32(smem) + tid * 16;
    auto issue = [&](int tile, uint32_t stage) {
        const uint32_t st = ring + stage;
        const uint8_t* from = reinterpret_cast<const uint8_t*>(p.body) + ((size_t)tile * kTileVecs + tid) * 16;
        const int left = p.nv - tile * kTileVecs;
        if (left >= kTileVecs) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(st + q * kThreads * 16),
                             "l"(from + q * kThreads * 16)
                             : "memory");
        } else if (left > 0) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
                if (q * kThreads + tid < left)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(st + q * kThreads * 16),
                                 "l"(from + q * kThreads * 16)
                                 : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kStages; ++i) issue(i, i * kTileVecs * 16);

    if (tid == 0) s_count = s_work = 0;
    uint32_t tok = 0;
    if (a.logprob && part == 0 && tid == 0) tok = a.tokens[r];
    // the row's ragged ends, one element per thread: its index, or -1
    int ragged = -1;
    if (part == 0 && tid < p.first) ragged = tid;
    if (tid >= 32 && p.first + nv * kN + tid - 32 < p.hi) ragged = p.first + nv * kN + tid - 32;

    // ---- this thread's share: sums, largest element, the pieces' maxima
    Sums s{-INFINITY, 0.0f, 0.0f};
    if (ragged >= 0) {
        const float x = to_f32(p.row[ragged]);
        raise(s, x, k);
        float2 z = f2(0.0f), y = f2(0.0f);
        add_two(z, y, x, -INFINITY, f2(-base_of(s.m)), f2(k));
        s.z += z.x;
        s.y += y.x;
    }
    float best = s.m, piece = -INFINITY;
    int left = per_slot, slot = tid;  // tiles left of the piece, its place in slot_max
    uint32_t stage = 0;
    auto consume = [&](int tile, auto whole) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        const uint8_t* st = smem + stage + tid * 16;
        float x[kVecs * kN];
#pragma unroll
        for (int q = 0; q < kVecs; ++q)
            unpack(p.row, *reinterpret_cast<const uint4*>(st + q * kThreads * 16), x + q * kN);
        if constexpr (!decltype(whole)::value) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
                if (tile * kTileVecs + q * kThreads + tid >= nv) {
#pragma unroll
                    for (int e = 0; e < kN; ++e) x[q * kN + e] = -INFINITY;
                }
        } else {
            issue(tile + kStages, stage);  // the stage's values are in registers
            stage = stage == (kStages - 1) * kTileVecs * 16 ? 0 : stage + kTileVecs * 16;
        }
        // the maximum three at a time, in two chains
        float m = x[0], m1 = x[1];
#pragma unroll
        for (int i = 2; i + 3 < kVecs * kN; i += 4) {
            m = max3(m, x[i], x[i + 1]);
            m1 = max3(m1, x[i + 2], x[i + 3]);
        }
        m = max3(max3(m, m1, piece), x[kVecs * kN - 2], x[kVecs * kN - 1]);
        piece = m;
        // the sums at the new maximum (a reference below it would cost the entropy of a peaked row its
        // digits: ln Z and Y / Z would both be large); -inf - -inf and -inf * 0 become factors of 0
        const float top = fmaxf(s.m, m), d = fmaxf((s.m - top) * k, -200.0f), f = ex2_approx(d);
        s.m = top;
        s.y = f * fmaf(d, s.z, s.y);
        s.z *= f;
        const float2 minus_m = f2(-base_of(s.m));
        float2 z = f2(0.0f), y = f2(0.0f);
#pragma unroll
        for (int i = 0; i < kVecs * kN; i += 2) add_two(z, y, x[i], x[i + 1], minus_m, f2(k));
        s.z += z.x + z.y;
        s.y += y.x + y.y;
        if (--left == 0 || tile + 1 == tiles) {
            slot_max[slot] = piece;
            best = fmaxf(best, piece);
            piece = -INFINITY;
            left = per_slot;
            slot += kThreads;
        }
    };
    for (int tile = 0; tile < whole_tiles; ++tile) consume(tile, std::true_type{});
    if (whole_tiles < tiles) consume(whole_tiles, std::false_type{});
    float tok_x = 0.0f;
    if (tok < (uint32_t)a.V && a.logprob && part == 0 && tid == 0) tok_x = to_f32(p.row[tok]);

    // ---- the block's n best as a list, its sums in s_part
    const int want = min(a.n_top, p.hi - p.lo);
    // adds every element with key > bound (or >= if ties) to the list
    auto gather = [&](uint32_t bound, bool ties) {
        const float floor = bound ? key_value(bound) : -INFINITY;
        const bool ge = ties || bound == 0, nan = ties && bound == 0;
        auto reaches = [&](float x) { return ge ? x >= floor || (nan && x != x) : x > floor; };
        auto offer = [&](float x, int i) {
            if (!reaches(x)) return;
            const int at = atomicAdd(&s_count, 1);
            if (at < kList) list[at] = full_key(order_key(x), i);
        };
        if (nan || reaches(best)) {
            for (int i = 0; i * per_slot < tiles; ++i)
                if (nan || reaches(slot_max[i * kThreads + tid]))
                    work[atomicAdd(&s_work, 1)] = (uint16_t)(i * kThreads + tid);
        }
        if (ragged >= 0) offer(to_f32(p.row[ragged]), ragged);
        __syncthreads();
        // eight lanes read a piece's vectors
        const int n = s_work;
        for (int i = tid >> 3; i < n; i += kThreads / 8) {
            const int at = work[i], first = at / kThreads * per_slot;
            for (int j = tid & 7; j < per_slot * kVecs; j += 8) {
                const int v = (first + j / kVecs) * kTileVecs + (j % kVecs) * kThreads + at % kThreads;
                if (v >= nv) continue;
                float x[kN];
                unpack(p.row, __ldg(reinterpret_cast<const uint4*>(p.body + (size_t)v * kN)), x);
#pragma unroll
                for (int e = 0; e < kN; ++e) offer(x[e], p.first + v * kN + e);
            }
        }
    };
    auto post_sums = [&] {
        s = warp_join(s, k, 32);
        if (lane == 0) s_part[warp] = s;
    };
    uint32_t bound = 0;
    if (a.n_top) {
        // each warp keeps a few more than its share of its threads' maxima; the n-th largest of all
        // that are kept is a bound which n elements reach
        const int full_warps = min(kWarps, nv / 32);  // warps whose every lane has data
        const int keep = full_warps ? min(32, (a.n_top + full_warps - 1) / full_warps + 2) : 0;
        const int kept = full_warps * keep;
        if (tid < 4) s_bound[kept + tid] = 0;  // read with the last ones, below all
        uint32_t key = order_key(best);
        for (int i = 0; i < keep; ++i) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, key);
            const uint32_t who = __ballot_sync(0xffffffffu, key == top);
            if (lane == __ffs(who) - 1) {
                if (warp < full_warps) s_bound[warp * keep + i] = key;
                key = 0;
            }
        }
        __syncthreads();
        if (kept >= a.n_top) {
            for (int i = lane; i < (kept + 31) / 32 * 32; i += 32) {
                const uint32_t v = i < kept ? s_bound[i] : 0u;
                int rank = 0;
#pragma unroll 2
                for (int j = 0; j < kept; j += 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(s_bound + j);
                    rank += (x.x > v) + (x.y > v) + (x.z > v) + (x.w > v);
                    rank += (x.x == v && j < i) + (x.y == v && j + 1 < i) + (x.z == v && j + 2 < i) + (x.w == v && j + 3 < i);
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, i < kept && rank == a.n_top - 1);
                if (hit) {
                    bound = __shfl_sync(0xffffffffu, v, __ffs(hit) - 1);
                    break;
                }
            }
        }
    } else {
        __syncthreads();
    }
    int c = 0;
    if (a.n_top) {
        bool ties = true;
        for (;;) {
            gather(bound, ties);
            if (ties) post_sums();
            __syncthreads();
            c = s_count;
            // complete: everything from the bound on, or everything above it
            if (c <= kList && (!ties || c >= want)) break;
            if (c > kList && !ties) {  // a higher bound: the want-th best of those listed
                rank_list<kThreads>(list, kList, [&](int rank, unsigned long long key) {
                    if (rank == want - 1) s_raise = key;
                });
                __syncthreads();
                bound = (uint32_t)(s_raise >> 32);
            } else if (c < want) {  // NaN entries among the best: below everything else
                bound = 0;
            }
            ties = false;
            __syncthreads();
            if (tid == 0) s_count = s_work = 0;
            __syncthreads();
        }
        // the first elements equal to the bound, in index order
        const int need = want - c;
        int seen = 0;
        for (int base = p.lo; base < p.hi && seen < need; base += kThreads) {
            const int i = base + tid;
            const bool tie = i < p.hi && order_key(to_f32(p.row[i])) == bound;
            const uint32_t bal = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) s_warp[warp] = __popc(bal);
            __syncthreads();
            int before = seen + __popc(bal & ((1u << lane) - 1));
            for (int j = 0; j < kWarps; ++j) {
                if (j < warp) before += s_warp[j];
                seen += s_warp[j];
            }
            if (tie && before < need) list[c + before] = full_key(bound, i);
            __syncthreads();
        }
        if (need > 0) c += min(seen, need);
    } else {
        post_sums();
        __syncthreads();
    }
    if (cluster == 1 && warp > 0 && warp * 32 >= c) return;  // nothing to write
    s = warp_join(s_part[lane % kWarps], k, kWarps);
    s.m = __shfl_sync(0xffffffffu, s.m, 0);
    s.z = __shfl_sync(0xffffffffu, s.z, 0);
    s.y = __shfl_sync(0xffffffffu, s.y, 0);

    // ---- over the cluster (which has one row)
    if (cluster > 1) {
        unsigned long long* mine = reinterpret_cast<unsigned long long*>(smem + S::kInboxOfs);
        rank_list<kThreads>(list, c, [&](int rank, unsigned long long key) {
            if (rank < want) mine[rank] = key;
        });
        __syncthreads();
        cluster_wait();  // all blocks have started
        if (part != 0) {
            const uint32_t box = map_to_first(smem_u32(smem + S::kInboxOfs + part * kInboxStride));
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
        c = want;
        for (int i = tid; i < want; i += kThreads) list[i] = mine[i];
        for (int q = 1; q < cluster; ++q) {
            const uint8_t* box = smem + S::kInboxOfs + q * kInboxStride;
            const float* f = reinterpret_cast<const float*>(box + kMaxTop * 8);
            s = join(s, Sums{f[0], f[1], f[2]}, k);
            const int n = __float_as_int(f[3]);
            for (int i = tid; i < n; i += kThreads) list[c + i] = reinterpret_cast<const unsigned long long*>(box)[i];
            c += n;
        }
        __syncthreads();
    }

    // NaN and +inf have made Z NaN; Z is 0 only for a row of -inf
    const float log_z = logf(s.z);
    auto lp = [&](float x) {
        if (log_z != log_z) return log_z;
        const float d = 0.5f * x - 0.5f * base_of(s.m);  // halves: the difference may pass the largest f32
        return d == -INFINITY ? d : fmaf(d, 2.0f * a.inv_t, -log_z);
    };
    if (tid == 0) {
        if (a.logprob) {
            if (tok >= (uint32_t)a.V) atomicCAS(a.err, 0, kErrToken);
            a.logprob[r] = tok < (uint32_t)a.V ? lp(tok_x) : __int_as_float(0x7fc00000);
        }
        if (a.entropy) a.entropy[r] = s.z == 0.0f ? 0.0f : log_z - kLn2 * (s.y / s.z);
    }
    if (a.n_top)
        rank_list<kThreads>(list, c, [&](int rank, unsigned long long key) {
            if (rank >= a.n_top) return;
            a.top_tokens[(size_t)r * a.n_top + rank] = ~(uint32_t)key;
            a.top_logprobs[(size_t)r * a.n_top + rank] = lp(key_value((uint32_t)(key >> 32)));
        });
}

// Blocks per row: enough for `want` blocks, as long as each keeps a tile's worth.
int log_cluster_of(const TokenLogprobsArgs& a, int elt, int want) {
    const int per_tile = Block<256, 2>::kTileVecs * 16 / elt;
    int c = 0;
    while (1 << c < kMaxCluster && ((long long)a.M << c) < want && a.V >> (c + 1) >= per_tile) ++c;
    return c;
}

template <typename T, int kStages>
cudaError_t launch_wide(const TokenLogprobsArgs& a, int log_cluster, cudaStream_t s) {
    static SmemAttr attr;
    using S = Block<256, kStages>;
    const cudaError_t e = ensure_smem(attr, token_logprobs_kernel<T, 256, kStages>, S::kSmemCluster);
    if (e != cudaSuccess) return e;
    return launch_dependent(token_logprobs_kernel<T, 256, kStages>, dim3((unsigned)a.M << log_cluster), 256,
                            log_cluster ? S::kSmemCluster : S::kSmemOne, 1 << log_cluster, s, a, log_cluster);
}

template <typename T>
cudaError_t launch_typed(const TokenLogprobsArgs& a, int sm_count, cudaStream_t s) {
    // many short rows: a block's time is mostly its steps of selection, so small blocks, sixteen to
    // an SM (4096 rows of 1000 f32: 40.4 us with 256 threads, 12.8 with 64)
    if ((size_t)a.V * sizeof(T) <= kShortRow && a.M > 4 * sm_count) {
        return launch_dependent(token_logprobs_kernel<T, 64, 2>, dim3((unsigned)a.M), 64, Block<64, 2>::kSmemOne, 1, s,
                                a, 0);
    }
    // Rows whose clusters fill the SMs once but not twice over: one wave of blocks, each with twice the
    // bytes in flight, against two waves' worth of blocks with the shorter ring (128256 f32 each: 19
    // rows 11.0 -> 9.8 us, 64 rows 14.1 -> 11.5, 140 rows 21.9 -> 20.0).  With fewer blocks the longer
    // ring is of no use (8 rows 8.5 us, 8.8 with it), with one row per block it fits less often.
    // Clusters of 8 find two blocks' room per SM only within an SM group: past 30 or so of them a second
    // wave forms (32 rows 13.6 us), and clusters of 4 are taken (11.1).
    int c = log_cluster_of(a, (int)sizeof(T), sm_count);
    if (c > 0 && a.M << c >= sm_count) {
        if (c == 3 && (a.M << c) * 8 > 13 * sm_count) c = 2;
        return launch_wide<T, 4>(a, c, s);
    }
    return launch_wide<T, 2>(a, log_cluster_of(a, (int)sizeof(T), 2 * sm_count), s);
}

}  // namespace

cudaError_t launch_token_logprobs(const TokenLogprobsArgs& a, int sm_count, cudaStream_t s) {
    if (a.dtype == VELO_ELEM_F32) return launch_typed<float>(a, sm_count, s);
    if (a.dtype == VELO_ELEM_F16) return launch_typed<__half>(a, sm_count, s);
    return launch_typed<__nv_bfloat16>(a, sm_count, s);
}

}  // namespace velo
