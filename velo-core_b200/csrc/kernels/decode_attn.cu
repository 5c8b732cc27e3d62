// decode_attn.cu -- attention of one query token per sequence over the paged
// cache (velo_cuda_decode_attention).
//
// s_j = scale q.k_j, p = softmax(s), out = sum p_j v_j: every K and V byte is used
// once per KV head by its few query heads (4 flop per element and head), so HBM
// bounds it and the matrix work only has to stay out of the way.
//
// Work: the batch is one list of units -- a unit is a step of 16 (f16), 32 (int8)
// or 8 (f32) tokens of one item, an item a (sequence, KV head, tile of query
// heads) -- cut into equal ranges, one per block, two blocks per SM, whatever the
// lengths are (and a tail of short ranges, for balance; decode_cut.cuh).  An item that a cut runs
// through leaves partial states (max, sum, unnormalised output) in the workspace,
// which the join kernel, launched as a programmatic dependent, adds in order: no
// atomics, repeatable bits.  Short items are not cut (the cut moves to their
// start), so a batch of short contexts pays no join.  What it pays is each item's start and
// end, 1.3 us of an SM (256 x 32 tokens, 32/8 heads f16: 25.3 us), so the next item's q is on
// its way while the warps' states of the last one are joined (5 us more without).
//
// A block's four warps take the units of its range in turn.  Each warp streams
// its own units through a private ring of 8 KB (head_dim 128) stages filled by
// 16-byte cp.async (three stages: 96 KB in flight per block), so no block-wide
// barrier stands between the loads and the arithmetic; tokens past the length are
// zero-filled, never read.  Query heads of a KV head are the columns of mma.sync
// tiles (m16n8k16; tcgen05's 128-row tiles would be 1/16 full at 8 heads a KV head).
//
//  The weights are held in f32 and enter P V as two f16 parts (value and remainder) in a
//   unit of the step's own largest weight of that head: 2^-22 of a weight, or 2^-39 of the
//   step's largest, is all that is lost, so many small weights beside a dominant one add up
//   as the f32 sum in the denominator does.  (In units of the reference, a weight 2^-25
//   below it would be 0.)  The step's sums are added to the output by f32 multiply-adds.
//   With at most 4 heads the parts share a tile: columns 0 - 3 and 4 - 7.
//  f16: K and V fragments by ldmatrix from XOR-swizzled rows.
//  int8: K fragments are 16 consecutive bytes per lane (the contraction order is free, q is
//   permuted to match), V is transposed in 16-bit units by ldmatrix.trans.  A byte plus 128 in
//   the low bits of an f16 is a subnormal, exact as an operand (one LOP3 or a shift and one
//   for two values); 128 times the sum of q, and of the weights, comes off the results.  The
//   K scale multiplies the score and the V scale the weight.
//  f32: FFMA, a lane per (token, quarter of the head) for the scores and per 4 (2)
//   dimensions for the output.  (Exponentials are ex2.approx, 2^-22, in all forms.)
//
// Measured on a B200 against 6552 GB/s, device time back to back: 64 sequences of 3900 - 4290
// f16 tokens, 64/8 heads, 174.6 us (0.94); one of 100003 tokens 73.8 us (0.85: start-up and
// join); 128 ragged INT8 sequences, 32/8 heads, 229 us (0.78) at the 1500 MHz that the power cap
// leaves, 201 in a short burst; one of 203 tokens 6.7 us, which is latency: length,
// page and K/V reads in a row, four steps of a warp, the launch.  The step's own unit of the
// weights costs 1.6 us of the 174.6 and 0.2 of the 6.7.
#include <algorithm>
#include <type_traits>

#include "common/elem.cuh"
#include "common/pdl.cuh"
#include "common/sm100.cuh"
#include "common/smem_attr.cuh"
#include "kernels/decode_cut.cuh"
#include "kernels/decode_ops.h"
#include "velo_cuda.h"

namespace velo {
namespace {

using sm100::ex2_approx;
using sm100::smem_u32;

constexpr int kErrSeqLen = 0x6211, kErrPage = 0x6212;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kRing = 64;  // unit descriptions per warp

constexpr int bytes_of(int kv) { return kv == VELO_KV_F16 ? 2 : kv == VELO_KV_INT8 ? 1 : 4; }

// Shared memory of a block; the lengths and the prefix sums follow.
template <int KV, int D, int R>
struct Layout {
    static constexpr int kTok = tokens_of(KV);
    static constexpr int kRow = D * bytes_of(KV);               // bytes of a token's K or V
    static constexpr int kHalf = kTok * kRow;                   // K, then V
    static constexpr int kStage = 2 * kHalf + (KV == VELO_KV_INT8 ? 4 * kTok : 0);  // + scales
    static constexpr int kStages = (blocks_per_sm(KV, R) == 3 ? 2 : 3) * (128 / D);
    static constexpr int kJoinUnits = join_units(KV, D);
    static constexpr int kRings = kWarps * kStages * kStage;
    static constexpr int kStats = kRings + kWarps * kRing * 16;
    static constexpr int kQ = kStats + 3 * kWarps * 16 * 4;     // f32: q, and each warp's weights
    static constexpr int kP = kQ + (KV == VELO_KV_F32 ? 8 * D * 4 : 0);
    static constexpr int kLens = kP + (KV == VELO_KV_F32 ? kWarps * 72 * 4 : 0);
};

// A partial state: rows x (max, sum), then rows x D of output.
__host__ __device__ inline size_t slot_floats(int rows, int D) { return (size_t)rows * (D + 2); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float lds_half(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return __half2float(__ushort_as_half(v));
}
// The 8 x 8 matrix of 16-bit elements a warp holds (lane 4 row + t: columns 2t,
// 2t + 1), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// The largest over the lanes of a head's scores (those with the same lane % 4).
__device__ __forceinline__ float max_of_tokens(float x) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

// Two f32 as a pair of 16-bit parts and the pair of their remainders.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
}
// The even (odd) bytes of w, int8, plus 128 and in units of 2^-24, as an f16 pair: a
// byte in the lowest bits of a f16 is a subnormal, which the tensor cores multiply
// exactly.  The 128 comes off the sums instead of every element.
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return (w & 0x00ff00ffu) ^ 0x00800080u; }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return even_bytes(w >> 8); }

// KV: velo_kv_dtype; D: head_dim; R: tiles of 8 query heads per item (0: half a tile).
template <int KV, int D, int kTiles>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(KV, kTiles)) decode_attn_kernel(const DecodeAttnArgs a,
                                                                                     const Plan plan) {
    using L = Layout<KV, D, kTiles>;
    using Act = typename std::conditional<KV == VELO_KV_F32, float, __half>::type;
    constexpr bool kPair = kTiles == 0;  // columns 4 .. 7 hold remainders
    constexpr int R = kPair ? 1 : kTiles, kTok = L::kTok, S = L::kStages, kRows = rows_of(kTiles);
    extern __shared__ __align__(128) uint8_t smem[];
    dependent_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int c = blockIdx.x, Hkv = a.kv.n_kv, Hq = a.Hq;
    const int per_seq = Hkv * plan.tiles;
    float* stat_m = reinterpret_cast<float*>(smem + L::kStats);  // [warp][16]
    float* stat_l = stat_m + kWarps * 16;
    int* stat_buf = reinterpret_cast<int*>(stat_l + kWarps * 16);
    int* lens = reinterpret_cast<int*>(smem + L::kLens);
    int* pre = lens + a.B;
    __shared__ int s_warp[kWarps], s_long[kWarps], s_filled[kWarps];
    int4* desc = static_cast<int4*>(a.ws);
    float* slots = reinterpret_cast<float*>(desc + plan.blocks);

    // lengths and units before each sequence
    auto length_of = [&](int b) {
        int n = a.seq_len[b];
        if (n < 0 || n > a.kv.max_pages * kPageTokens) {
            if (c == 0) atomicCAS(a.err, 0, kErrSeqLen);
            n = n < 0 ? 0 : a.kv.max_pages * kPageTokens;
        }
        return n;
    };
    auto running_sum = [&](int x) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    int total, longest, filled;
    if (a.B <= 32) {  // every warp by itself, all with the same results: no barrier
        const int n = lane < a.B ? length_of(lane) : 0, units = (n + kTok - 1) / kTok;
        const int x = running_sum(units * per_seq);
        if (lane < a.B) {
            lens[lane] = n;
            pre[lane] = x - units * per_seq;
        }
        total = __shfl_sync(0xffffffffu, x, 31);
        if (lane == 0) pre[a.B] = total;
        longest = __reduce_max_sync(0xffffffffu, units);
        filled = __popc(__ballot_sync(0xffffffffu, n > 0));
        __syncwarp();
    } else {
        const int per = (a.B + kThreads - 1) / kThreads, lo = min(tid * per, a.B), hi = min(lo + per, a.B);
        int sum = 0;
        longest = filled = 0;
        for (int b = lo; b < hi; ++b) {
            const int n = length_of(b), units = (n + kTok - 1) / kTok;
            lens[b] = n;
            pre[b] = sum;
            sum += units * per_seq;
            longest = max(longest, units);
            filled += n > 0;
        }
        const int x = running_sum(sum);
        longest = __reduce_max_sync(0xffffffffu, longest);
        filled = __reduce_add_sync(0xffffffffu, filled);
        if (lane == 31) {
            s_warp[warp] = x;
            s_long[warp] = longest;
            s_filled[warp] = filled;
        }
        __syncthreads();
        int before = x - sum;
        longest = filled = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_warp[w];
            longest = max(longest, s_long[w]);
            filled += s_filled[w];
        }
        for (int b = lo; b < hi; ++b) pre[b] += before;
        if (tid == kThreads - 1) pre[a.B] = before + sum;
        __syncthreads();
        total = pre[a.B];
    }
    const Cut list = cut_list(plan, total, filled * per_seq, longest, L::kJoinUnits);

    // sequences without tokens
    for (int b = c; b < a.B; b += gridDim.x) {
        if (lens[b]) continue;
        for (int i = tid; i < Hq * D; i += kThreads) static_cast<Act*>(a.out)[(size_t)b * Hq * D + i] = (Act)0.0f;
        if (a.lse)
            for (int i = tid; i < Hq; i += kThreads) a.lse[(size_t)b * Hq + i] = -INFINITY;
    }
    if (c >= list.blocks()) {
        if (tid == 0) desc[c] = make_int4(-1, 0, 0, 0);
        return;
    }
    const int edge = lane < 2 ? cut_at<kTok>(pre, lens, a.B, list, L::kJoinUnits, c + lane) : 0;
    const int u0 = __shfl_sync(0xffffffffu, edge, 0), u1 = __shfl_sync(0xffffffffu, edge, 1);

    // ---- this warp's stream of units
    const int n_w = max(0, (u1 - u0 - warp + kWarps - 1) / kWarps);
    uint4* ring = reinterpret_cast<uint4*>(smem + L::kRings) + warp * kRing;
    const uint32_t stage0 = smem_u32(smem + warp * S * L::kStage);
    auto describe = [&](int j0) {  // the units j0 .. j0 + 31: pages, head, tokens present
        const int j = j0 + lane;
        if (j >= n_w) return;
        const int u = u0 + warp + kWarps * j;
        const Item x = item_of<kTok>(pre, lens, a.B, u);
        const int first = (u - x.start) * kTok, left = lens[x.b] - first;
        const uint32_t* row = a.kv.page_table + (size_t)x.b * a.kv.max_pages + first / kPageTokens;
        uint4 e = make_uint4(row[0], 0, (uint32_t)(plan.tiles == 1 ? x.it : x.it / plan.tiles), left >= 32 ? ~0u : (1u << left) - 1);
        uint32_t low = kTok == 8 ? 0xffu : 0xffffu;
        e.w &= kTok == 32 ? ~0u : low;
        if (e.x >= (uint32_t)a.kv.pool_pages) {
            atomicCAS(a.err, 0, kErrPage);
            e.x = 0;
            e.w &= ~low;
        }
        if (kTok == 32 && left > 16) {
            e.y = row[1];
            if (e.y >= (uint32_t)a.kv.pool_pages) {
                atomicCAS(a.err, 0, kErrPage);
                e.y = 0;
                e.w &= 0xffffu;
            }
        }
        if (kTok == 8) e.y = first % kPageTokens;  // the page's half
        ring[j % kRing] = e;
    };
    // An instruction copies 512 bytes: 32 chunks of kPer rows.  Chunk c of row r lies at
    // c ^ swizzle(r) of its row; the swizzles split into a part of the instruction
    // and one of the lane.
    constexpr int kChunks = L::kRow / 16, kPer = 32 / kChunks, kIts = kTok / kPer;
    auto k_swizzle = [](int row) {
        return KV == VELO_KV_F16 ? row & 7 : KV == VELO_KV_INT8 && D == 64 ? 0 : (row & 1) << 2;
    };
    auto v_swizzle = [](int row) {
        return KV == VELO_KV_F32 ? 0 : KV == VELO_KV_INT8 && D == 64 ? (row >> 1) & 3 : row & 7;
    };
    const uint32_t k_dst = lane / kChunks * L::kRow + (((lane % kChunks) ^ k_swizzle(lane / kChunks)) << 4);
    const uint32_t v_dst = lane / kChunks * L::kRow + (((lane % kChunks) ^ v_swizzle(lane / kChunks)) << 4);
    constexpr uint32_t kFull = kTok == 32 ? ~0u : (1u << kTok) - 1;
    auto issue = [&](int j) {
        if (j < n_w) {
            if (j % 32 == 0) {
                describe(j);
                __syncwarp();
            }
            const uint4 e = ring[j % kRing];
            const uint32_t st = stage0 + (j % S) * L::kStage;
            const size_t block0 = ((size_t)e.x * Hkv + e.z) * kPageTokens + (kTok == 8 ? e.y : 0);
            const size_t block1 = kTok == 32 ? ((size_t)e.y * Hkv + e.z) * kPageTokens - 16 : block0;
            const uint8_t* k0 = static_cast<const uint8_t*>(a.kv.k_pool) + block0 * L::kRow + lane * 16;
            const uint8_t* v0 = static_cast<const uint8_t*>(a.kv.v_pool) + block0 * L::kRow + lane * 16;
            const uint8_t* k1 = static_cast<const uint8_t*>(a.kv.k_pool) + block1 * L::kRow + lane * 16;
            const uint8_t* v1 = static_cast<const uint8_t*>(a.kv.v_pool) + block1 * L::kRow + lane * 16;
            auto copy = [&](auto whole) {
#pragma unroll
                for (int i = 0; i < kIts; ++i) {
                    const bool second = kTok == 32 && i * kPer >= 16;
                    const uint32_t kd = st + i * 512 + (k_dst ^ (k_swizzle(i * kPer) << 4));
                    const uint32_t vd = st + L::kHalf + i * 512 + (v_dst ^ (v_swizzle(i * kPer) << 4));
                    const uint8_t *ks = (second ? k1 : k0) + i * 512, *vs = (second ? v1 : v0) + i * 512;
                    if constexpr (decltype(whole)::value) {
                        cp_async16(kd, ks);
                        cp_async16(vd, vs);
                    } else {  // rows past the length are zero-filled
                        const int n = (e.w >> (i * kPer + lane / kChunks)) & 1 ? 16 : 0;
                        cp_async16(kd, ks, n);
                        cp_async16(vd, vs, n);
                    }
                }
            };
            if (e.w == kFull)
                copy(std::true_type{});
            else
                copy(std::false_type{});
            if (KV == VELO_KV_INT8 && lane < 8) {  // scales: K of both pages, V of both pages
                const int pg = (lane >> 1) & 1, half = lane & 1;
                const size_t at = (pg ? block1 + 16 : block0) + half * 8;
                const int n = (e.w >> (pg * 16 + half * 8)) & 0xff ? 16 : 0;
                cp_async16(st + 2 * L::kHalf + lane * 16, (lane < 4 ? a.kv.k_scale : a.kv.v_scale) + at, n);
            }
        }
        cp_async_commit();
    };
    for (int j = 0; j < S; ++j) issue(j);

    const float scale = a.scale * kLog2e;
    constexpr int kH = KV == VELO_KV_F32 ? 1 : R;
    uint32_t qb[kH][KV == VELO_KV_F32 ? 1 : D / 16][2];  // q as B fragments: head 8r + g
    // reads an item's q; the next item's is on its way while the warps' states are joined
    auto load_q = [&](int b, int hk, int tile) {
        const int nh = min(kRows, plan.group - tile * kRows);
        const Act* qp = static_cast<const Act*>(a.q) + (size_t)b * a.ldq + (size_t)(hk * plan.group + tile * kRows) * D;
        if constexpr (KV != VELO_KV_F32) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int row = kPair ? g & 3 : 8 * r + g;
                const Act* qr = qp + (size_t)row * D;
                // the dimensions a lane holds of contraction step ks: ldmatrix's own order for f16,
                // 4 consecutive ones for int8 (16 of four steps: two loads)
                if constexpr (KV == VELO_KV_F16) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            qb[r][ks][i] =
                                row < nh ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8 * i + 2 * t) : 0u;
                } else {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const uint4 v = row < nh ? *reinterpret_cast<const uint4*>(qr + 64 * (i / 2) + 16 * t + 8 * (i % 2))
                                                 : make_uint4(0, 0, 0, 0);
                        qb[r][2 * i][0] = v.x;
                        qb[r][2 * i][1] = v.y;
                        qb[r][2 * i + 1][0] = v.z;
                        qb[r][2 * i + 1][1] = v.w;
                    }
                }
            }
        }
    };
    int j = 0;
    int4 open = make_int4(-1, 0, 0, 0);
    Item x{};
    int hk = 0, tile = 0;  // of the item
    if (u0 < u1) {
        x = item_of<kTok>(pre, lens, a.B, u0);
        hk = plan.tiles == 1 ? x.it : x.it / plan.tiles;
        tile = x.it - hk * plan.tiles;
        load_q(x.b, hk, tile);
    }
    for (int seg = u0; seg < u1;) {
        const int end = x.start + x.units, seg_end = min(end, u1);
        const int h0 = hk * plan.group + tile * kRows, nh = min(kRows, plan.group - tile * kRows);

        // ---- running state.  Tensor cores: scores and output are held transposed (keys or
        // dimensions x heads), so a lane has heads 8r + 2t + {0, 1}; f32: heads 2t + {0, 1} of
        // its token.  m is the reference of the weights, at most 2^8 below the largest.
        float m[kH][2], l[kH][2];
#pragma unroll
        for (int r = 0; r < kH; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[r][e] = -INFINITY;
                l[r][e] = 0.0f;
            }
        constexpr int kN = KV == VELO_KV_F32 ? 1 : D / 16;      // output tiles of 16 dimensions
        float o[kH][kN][4] = {};
        constexpr int kO = KV == VELO_KV_F32 ? D / 32 : 1;      // dimensions per lane
        float of[KV == VELO_KV_F32 ? 8 : 1][kO] = {};
        if constexpr (KV == VELO_KV_F32) {
            const Act* qp = static_cast<const Act*>(a.q) + (size_t)x.b * a.ldq + (size_t)h0 * D;
            float* qs = reinterpret_cast<float*>(smem + L::kQ);
            for (int i = tid; i < 8 * D; i += kThreads) qs[i] = i / D < nh ? to_f32(qp[i]) : 0.0f;
            __syncthreads();
        }
        if constexpr (KV == VELO_KV_INT8) {  // the even, then the odd ones of 4 consecutive dimensions
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t lo = qb[r][ks][0], hi = qb[r][ks][1];
                    qb[r][ks][0] = __byte_perm(lo, hi, 0x5410);
                    qb[r][ks][1] = __byte_perm(lo, hi, 0x7632);
                }
        }
        // INT8: the scores carry 128 times the sum of q, which comes off each of them.  Their f32 sums
        // are then as exact as those of a K row whose values all have its maximum's size: 2^-24 of
        // sum |q| max|k| a step, far below the page's own rounding (max|k| / 127).
        float q128[kH][2];
        if constexpr (KV == VELO_KV_INT8) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sum = 0.0f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qb[r][ks][i]));
                        sum += f.x + f.y;
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // head 8r + g
#pragma unroll
                for (int e = 0; e < 2; ++e) q128[r][e] = 128.0f * __shfl_sync(0xffffffffu, sum, 4 * (2 * t + e));
            }
        }
        bool pending = false;
        for (; j < n_w && u0 + warp + kWarps * j < seg_end; ++j) {
            if (pending) issue(j - 1 + S);
            cp_async_wait<S - 1>();
            __syncwarp();
            const uint32_t st = stage0 + (j % S) * L::kStage;
            const uint32_t present = ring[j % kRing].w;
            if constexpr (KV != VELO_KV_F32) {
                // ---- scores of 16 kt + {g, 8 + g}: two accumulators each, to halve the chain
                constexpr int kT = kTok / 16;
                float s[kT][R][4];
                {
                    float sum[2][kT][R][4];
                    if constexpr (KV == VELO_KV_F16) {
                        const int r8 = lane & 7, mi = lane >> 3;
                        const uint32_t kb = st + ((mi & 1) * 8 + r8) * L::kRow;
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            uint32_t kf[4];
                            ldmatrix_x4(kf, kb + (((2 * ks + (mi >> 1)) ^ r8) << 4));
#pragma unroll
                            for (int r = 0; r < R; ++r) {
                                if (ks < 2)
                                    mma_f16_zero(sum[ks][0][r], kf, qb[r][ks][0], qb[r][ks][1]);
                                else
                                    mma_f16(sum[ks & 1][0][r], kf, qb[r][ks][0], qb[r][ks][1]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
#pragma unroll
                            for (int kt = 0; kt < kT; ++kt) {
                                uint32_t w[2][4];  // 16 bytes of tokens g and 8 + g
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const int row = kt * 16 + 8 * i + g, ch = (4 * h + t) ^ (D == 128 ? (row & 1) << 2 : 0);
                                    const uint4 v = lds128(st + row * L::kRow + ch * 16);
                                    w[i][0] = v.x;
                                    w[i][1] = v.y;
                                    w[i][2] = v.z;
                                    w[i][3] = v.w;
                                }
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t kf[4] = {even_bytes(w[0][i]), even_bytes(w[1][i]),
                                                            odd_bytes(w[0][i]), odd_bytes(w[1][i])};
#pragma unroll
                                    for (int r = 0; r < R; ++r) {
                                        if (h == 0 && i < 2)
                                            mma_f16_zero(sum[i][kt][r], kf, qb[r][i][0], qb[r][i][1]);
                                        else
                                            mma_f16(sum[i & 1][kt][r], kf, qb[r][4 * h + i][0], qb[r][4 * h + i][1]);
                                    }
                                }
                            }
                    }
#pragma unroll
                    for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[kt][r][e] = sum[0][kt][r][e] + sum[1][kt][r][e];
                }
                // ---- weights: element 2i + e is token 16 kt + 8i + g, head 8r + 2t + e
                float vs[kT][2];
#pragma unroll
                for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float f = scale;
                        if constexpr (KV == VELO_KV_INT8) {
                            const uint32_t at = st + 2 * L::kHalf + (kt * 16 + 8 * i + g) * 2;
                            f *= lds_half(at);
                            vs[kt][i] = lds_half(at + 2 * kTok);
                        }
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& x = s[kt][r][2 * i + e];
                                x = (KV == VELO_KV_INT8 ? fmaf(x, 16777216.0f, -q128[r][e]) : x) * f;
                            }
                    }
                // one rarely taken branch: a ragged step or a new reference
                bool adjust = present != kFull;
                float top[R][2];
                auto largest = [&] {  // of this lane's scores
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            top[r][e] = fmaxf(s[0][r][e], s[0][r][2 + e]);
#pragma unroll
                            for (int kt = 1; kt < kT; ++kt) top[r][e] = fmaxf(top[r][e], fmaxf(s[kt][r][e], s[kt][r][2 + e]));
                        }
                };
                largest();
#pragma unroll
                for (int r = 0; r < R; ++r) adjust |= top[r][0] > m[r][0] + 8.0f || top[r][1] > m[r][1] + 8.0f;
                if (__any_sync(0xffffffffu, adjust)) {
                    if (present != kFull) {
#pragma unroll
                        for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                if (!((present >> (kt * 16 + 8 * i + g)) & 1)) {
                                    if constexpr (KV == VELO_KV_INT8) vs[kt][i] = 0.0f;
#pragma unroll
                                    for (int r = 0; r < R; ++r) s[kt][r][2 * i] = s[kt][r][2 * i + 1] = -INFINITY;
                                }
                        largest();
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float mn = fmaxf(m[r][e], max_of_tokens(top[r][e]));
                            const float alpha = mn == m[r][e] ? 1.0f : ex2_approx(m[r][e] - mn);
                            m[r][e] = mn;
                            l[r][e] *= alpha;
#pragma unroll
                            for (int n = 0; n < kN; ++n) {
                                o[r][n][e] *= alpha;
                                o[r][n][2 + e] *= alpha;
                            }
                        }
                }
                // ---- the weights in f32, for P V times the V scale, and each head's unit: the power of two
                // that brings the step's largest to 2^14 .. 2^15, so that the two f16 parts keep 2^-22 of a
                // weight, or 2^-39 of the step's largest one, however far below the reference all of them are
                float unit[R][2];  // then what undoes it (and, INT8, the values' 2^-24)
                {
                    float most[R][2] = {};
#pragma unroll
                    for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                        for (int r = 0; r < R; ++r)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float& x = s[kt][r][2 * i + e];
                                    x = ex2_approx(x - (m[r][e] == -INFINITY ? 0.0f : m[r][e]));
                                    l[r][e] += x;
                                    if constexpr (KV == VELO_KV_INT8) x *= vs[kt][i];
                                    most[r][e] = fmaxf(most[r][e], KV == VELO_KV_INT8 ? fabsf(x) : x);
                                }
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t up = min(268u - (__float_as_uint(max_of_tokens(most[r][e])) >> 23), 254u);
                            const float by = __uint_as_float(up << 23);
#pragma unroll
                            for (int kt = 0; kt < kT; ++kt) {
                                s[kt][r][e] *= by;
                                s[kt][r][2 + e] *= by;
                            }
                            unit[r][e] = __uint_as_float((254u - up + (KV == VELO_KV_INT8 ? 24u : 0u)) << 23);
                        }
                }
                // ---- the weights, as value and remainder, become B fragments by transposition; P V
                uint32_t hi[kT][R][2], lo[kT][R][2];  // kPair: hi has both
#pragma unroll
                for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t h, rest;
                            split_f16(s[kt][r][2 * i], s[kt][r][2 * i + 1], h, rest);
                            if constexpr (kPair) {
                                hi[kt][r][i] = transpose8x8(t < 2 ? h : rest);
                            } else {
                                hi[kt][r][i] = transpose8x8(h);
                                lo[kt][r][i] = transpose8x8(rest);
                            }
                        }
                auto add_tile = [&](float (&to)[4], const float (&y)[4], int r) {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float2 x = __ffma2_rn(make_float2(y[e], y[e + 1]), make_float2(unit[r][0], unit[r][1]),
                                                    make_float2(to[e], to[e + 1]));
                        to[e] = x.x;
                        to[e + 1] = x.y;
                    }
                };
                const int r8 = lane & 7, mi = lane >> 3, row0 = (mi >> 1) * 8 + r8;
                if constexpr (KV == VELO_KV_F16) {
                    const uint32_t vb = st + L::kHalf + row0 * L::kRow, flip = v_swizzle(row0);
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        uint32_t vf[4];
                        ldmatrix_x4_trans(vf, vb + (((2 * n + (mi & 1)) ^ flip) << 4));
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            float y[4];
                            mma_f16_zero(y, vf, hi[0][r][0], hi[0][r][1]);
                            if constexpr (!kPair) mma_f16(y, vf, lo[0][r][0], lo[0][r][1]);
                            add_tile(o[r][n], y, r);
                        }
                    }
                } else {
                    // the step's sums start from minus 128 times its weights, as the same products: what
                    // its values carry too much, never more than the step's own weights
                    const uint32_t minus128[4] = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
                    float bias[R][4];
#pragma unroll
                    for (int kt = 0; kt < kT; ++kt)
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            if (kt == 0)
                                mma_f16_zero(bias[r], minus128, hi[kt][r][0], hi[kt][r][1]);
                            else
                                mma_f16(bias[r], minus128, hi[kt][r][0], hi[kt][r][1]);
                            if constexpr (!kPair) mma_f16(bias[r], minus128, lo[kt][r][0], lo[kt][r][1]);
                        }
                    // transposed as 16-bit units, a register holds two dimensions of two tokens:
                    // row 8 half + g of tile n is dimension 32 (n / 2) + 16 half + 2 g + n % 2
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        float y[2][R][4];
#pragma unroll
                        for (int kt = 0; kt < kT; ++kt) {
                            const int row = kt * 16 + row0;
                            uint32_t w[4];
                            ldmatrix_x4_trans(w, st + L::kHalf + row * L::kRow + (((n + (mi & 1)) ^ v_swizzle(row)) << 4));
                            const uint32_t va[4] = {even_bytes(w[0]), even_bytes(w[1]), even_bytes(w[2]),
                                                    even_bytes(w[3])};
                            const uint32_t vo[4] = {odd_bytes(w[0]), odd_bytes(w[1]), odd_bytes(w[2]),
                                                    odd_bytes(w[3])};
#pragma unroll
                            for (int r = 0; r < R; ++r) {
                                if (kt == 0) {
                                    mma_f16_from(y[0][r], va, hi[kt][r][0], hi[kt][r][1], bias[r]);
                                    mma_f16_from(y[1][r], vo, hi[kt][r][0], hi[kt][r][1], bias[r]);
                                } else {
                                    mma_f16(y[0][r], va, hi[kt][r][0], hi[kt][r][1]);
                                    mma_f16(y[1][r], vo, hi[kt][r][0], hi[kt][r][1]);
                                }
                                if constexpr (!kPair) {
                                    mma_f16(y[0][r], va, lo[kt][r][0], lo[kt][r][1]);
                                    mma_f16(y[1][r], vo, lo[kt][r][0], lo[kt][r][1]);
                                }
                            }
                        }
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            add_tile(o[r][n], y[0][r], r);
                            add_tile(o[r][n + 1], y[1][r], r);
                        }
                    }
                }
            } else {
                // ---- f32 scores: token g, dimensions 16 i + 4 t .. + 3 of every head
                const float* qs = reinterpret_cast<const float*>(smem + L::kQ);
                float* pw = reinterpret_cast<float*>(smem + L::kP) + warp * 72;  // [token][head], then alpha[head]
                float s[8] = {};
#pragma unroll 2
                for (int i = 0; i < D / 16; ++i) {
                    const uint4 kw = lds128(st + g * L::kRow + (((4 * i + t) ^ ((g & 1) << 2)) << 4));
                    const float k0 = __uint_as_float(kw.x), k1 = __uint_as_float(kw.y), k2 = __uint_as_float(kw.z),
                                k3 = __uint_as_float(kw.w);
#pragma unroll
                    for (int h = 0; h < 8; ++h) {
                        const float4 qv = *reinterpret_cast<const float4*>(qs + h * D + 16 * i + 4 * t);
                        s[h] = fmaf(qv.x, k0, fmaf(qv.y, k1, fmaf(qv.z, k2, fmaf(qv.w, k3, s[h]))));
                    }
                }
                // reduce-scatter over the four lanes of a token: lane t keeps heads 2t, 2t + 1
                float a4[4], a2[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float give = t & 2 ? s[i] : s[4 + i], keep = t & 2 ? s[4 + i] : s[i];
                    a4[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float give = t & 1 ? a4[i] : a4[2 + i], keep = t & 1 ? a4[2 + i] : a4[i];
                    a2[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
                }
                bool moved = false;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float sv = (present >> g) & 1 ? a2[r] * scale : -INFINITY;
                    float mx = sv;
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    const float mn = fmaxf(m[0][r], mx), rf = mn == -INFINITY ? 0.0f : mn;
                    const float al = ex2_approx(m[0][r] - rf), p = ex2_approx(sv - rf);
                    moved |= mn != m[0][r];
                    m[0][r] = mn;
                    l[0][r] = l[0][r] * al + p;
                    pw[g * 8 + 2 * t + r] = p;
                    if (g == 0) pw[64 + 2 * t + r] = al;
                }
                __syncwarp();
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int h = 0; h < 8; ++h)
#pragma unroll
                        for (int e = 0; e < kO; ++e) of[h][e] *= pw[64 + h];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float4 pA = *reinterpret_cast<const float4*>(pw + k * 8);
                    const float4 pB = *reinterpret_cast<const float4*>(pw + k * 8 + 4);
                    const float p[8] = {pA.x, pA.y, pA.z, pA.w, pB.x, pB.y, pB.z, pB.w};
                    float v[4];
                    if constexpr (D == 128) {
                        const uint4 w = lds128(st + L::kHalf + k * L::kRow + lane * 16);
                        v[0] = __uint_as_float(w.x);
                        v[1] = __uint_as_float(w.y);
                        v[2] = __uint_as_float(w.z);
                        v[3] = __uint_as_float(w.w);
                    } else {
                        const uint2 w = lds64(st + L::kHalf + k * L::kRow + lane * 8);
                        v[0] = __uint_as_float(w.x);
                        v[1] = __uint_as_float(w.y);
                    }
#pragma unroll
                    for (int h = 0; h < 8; ++h)
#pragma unroll
                        for (int e = 0; e < kO; ++e) of[h][e] = fmaf(p[h], v[e], of[h][e]);
                }
            }
            __syncwarp();  // every lane has read the stage
            pending = true;
        }

        Item next = x;
        if (seg_end < u1) {
            if (x.it + 1 < per_seq) {
                ++next.it;
                next.start = end;
                if (++tile == plan.tiles) {
                    tile = 0;
                    ++hk;
                }
            } else {
                next = item_of<kTok>(pre, lens, a.B, end);  // the next sequence's first item
                hk = tile = 0;
            }
            load_q(next.b, hk, tile);
        }

        // ---- the item's end in this range: the warps' states into one.  A warp's output goes
        // into the stage it has just read, which is refilled after the join.
        const uint32_t buf = stage0 + ((j + S - 1) % S) * L::kStage;  // stage of unit j - 1
#pragma unroll
        for (int r = 0; r < kH; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], d);
                if (g == 0) {
                    stat_m[warp * 16 + 8 * r + 2 * t + e] = m[r][e];
                    stat_l[warp * 16 + 8 * r + 2 * t + e] = l[r][e];
                }
            }
        if (kPair && KV != VELO_KV_F32 && pending) {  // the remainders' columns join their heads
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[0][n][e] += __shfl_xor_sync(0xffffffffu, o[0][n][e], 2);
        }
        if (lane == 0) stat_buf[warp] = (int)(buf - smem_u32(smem));
        if (pending) {
            float* dst = reinterpret_cast<float*>(smem + (buf - smem_u32(smem)));
            if constexpr (KV == VELO_KV_F32) {
#pragma unroll
                for (int h = 0; h < 8; ++h)
#pragma unroll
                    for (int e = 0; e < kO; ++e) dst[h * D + lane * kO + e] = of[h][e];
            } else {
                // [head][fragment row], eights XORed with the head against bank conflicts
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int n = 0; n < kN; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!kPair || t < 2) dst[(8 * r + 2 * t + (e & 1)) * D + ((16 * n + 8 * (e >> 1) + g) ^ (t << 3))] = o[r][n][e];
            }
        }
        __syncthreads();
        const bool whole = seg == x.start && seg_end == end;
        const int slot = 2 * c + (seg == x.start ? 1 : 0);
        float* sp = slots + (size_t)slot * slot_floats(kRows, D);
        for (int i = tid; i < nh * (D / 2); i += kThreads) {
            const int row = i / (D / 2), d = i % (D / 2) * 2;
            float M = -INFINITY, Ls = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, stat_m[w * 16 + row]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float lw = stat_l[w * 16 + row];
                if (lw == 0.0f) continue;  // nothing from this warp (its buffer is in flight)
                const float f = ex2_approx(stat_m[w * 16 + row] - M);
                const float* src = reinterpret_cast<const float*>(smem + stat_buf[w]) + row * D;
                const int flip = KV == VELO_KV_F32 ? 0 : (row >> 1 & 3) << 3;
                float v0, v1;
                if constexpr (KV == VELO_KV_INT8) {  // d even: its tile is even, d + 1 has the same row of the next tile
                    const int at = (d & ~31) + (d >> 1 & 15);
                    v0 = src[at ^ flip];
                    v1 = src[(at + 16) ^ flip];
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(src + (d ^ flip));
                    v0 = v.x;
                    v1 = v.y;
                }
                Ls = fmaf(lw, f, Ls);
                y0 = fmaf(v0, f, y0);
                y1 = fmaf(v1, f, y1);
            }
            if (whole) {
                const float inv = Ls == 0.0f ? 0.0f : 1.0f / Ls;
                Act* op = static_cast<Act*>(a.out) + ((size_t)x.b * Hq + h0 + row) * D + d;
                if constexpr (KV == VELO_KV_F32)
                    *reinterpret_cast<float2*>(op) = make_float2(y0 * inv, y1 * inv);
                else
                    *reinterpret_cast<__half2*>(op) = __floats2half2_rn(y0 * inv, y1 * inv);
                if (d == 0 && a.lse)
                    a.lse[(size_t)x.b * Hq + h0 + row] = Ls == 0.0f ? -INFINITY : (M + log2f(Ls)) * kLn2;
            } else {
                *reinterpret_cast<float2*>(sp + 2 * kRows + row * D + d) = make_float2(y0, y1);
                if (d == 0) *reinterpret_cast<float2*>(sp + 2 * row) = make_float2(M, Ls);
            }
        }
        __syncthreads();
        if (pending) issue(j - 1 + S);
        if (!whole && seg == x.start)  // begins here, ends in a later block
            open = make_int4(x.b, x.it, list.block_of(end - 1), 0);
        seg = seg_end;
        x = next;
    }
    cp_async_wait<0>();
    if (tid == 0) desc[c] = open;
}

// Joins the partial states of the item that block x of the first kernel left
// open: slot 1 of that block, slot 0 of the following ones.  A block's warps are
// shared out over the `rows` query heads of its blockIdx.y; each of a head's warps
// takes every per-th state, eight at a time (maxima, sums and outputs in one round
// of reads, the running maximum as in the first kernel), and their results are
// added in order.
template <typename Act, int D, int kJoinWarps, int rows>
__global__ void __launch_bounds__(kJoinWarps * 32) decode_join_kernel(const DecodeAttnArgs a, const Plan plan,
                                                                      int item_rows) {
    __shared__ float acc[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps];
    dependent_wait();  // the first kernel is complete and visible
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int per = kJoinWarps / rows;
    const int row = blockIdx.y * rows + warp / per, part = warp % per;
    const int4* desc = static_cast<const int4*>(a.ws);
    const int4 it = desc[c];
    if (it.x < 0) return;
    const int hk = it.y / plan.tiles, tile = it.y % plan.tiles;
    const bool live = tile * item_rows + row < plan.group;
    const int head = hk * plan.group + tile * item_rows + row;
    const size_t step = slot_floats(item_rows, D);
    const float* first = reinterpret_cast<const float*>(desc + plan.blocks) + (size_t)(2 * c) * step;
    const int n = live ? it.z - c + 1 : 0;
    constexpr int kE = D / 32, kBatch = 8;
    float m = -INFINITY, l = 0.0f, x[kE] = {};
    for (int i0 = part; i0 < n; i0 += per * kBatch) {
        float2 ml[kBatch];
        float o[kBatch][kE];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int i = i0 + j * per;
            ml[j] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int e = 0; e < kE; ++e) o[j][e] = 0.0f;
            if (i < n) {
                const float* st = first + (i == 0 ? 1 : 2 * (size_t)i) * step;
                ml[j] = *reinterpret_cast<const float2*>(st + 2 * row);
                const float* p = st + 2 * item_rows + row * D + lane * kE;
                if constexpr (kE == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(p);
                    o[j][0] = v.x, o[j][1] = v.y, o[j][2] = v.z, o[j][3] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(p);
                    o[j][0] = v.x, o[j][1] = v.y;
                }
            }
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) top = fmaxf(top, ml[j].x);
        const float ref = top == -INFINITY ? 0.0f : top, alpha = ex2_approx(m - ref);
        m = top;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < kE; ++e) x[e] *= alpha;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float f = ex2_approx(ml[j].x - ref);
            l = fmaf(ml[j].y, f, l);
#pragma unroll
            for (int e = 0; e < kE; ++e) x[e] = fmaf(o[j][e], f, x[e]);
        }
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[warp][lane * kE + e] = x[e];
    __syncthreads();
    if (part != 0 || !live) return;
    float M = -INFINITY, L = 0.0f, y[kE] = {};
#pragma unroll
    for (int w = 0; w < per; ++w) M = fmaxf(M, s_m[warp + w]);
#pragma unroll
    for (int w = 0; w < per; ++w) {
        const float f = ex2_approx(s_m[warp + w] - (M == -INFINITY ? 0.0f : M));
        L = fmaf(s_l[warp + w], f, L);
#pragma unroll
        for (int e = 0; e < kE; ++e) y[e] = fmaf(acc[warp + w][lane * kE + e], f, y[e]);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    Act* out = static_cast<Act*>(a.out) + ((size_t)it.x * a.Hq + head) * D + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; ++e) out[e] = (Act)(y[e] * inv);
    if (lane == 0 && a.lse) a.lse[(size_t)it.x * a.Hq + head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

template <int KV, int D, int R>
cudaError_t launch_typed(const DecodeAttnArgs& a, int sm_count, cudaStream_t s) {
    using L = Layout<KV, D, R>;
    static SmemAttr attr;
    const int smem = L::kLens + (2 * a.B + 1) * 4;
    cudaError_t e = ensure_smem(attr, decode_attn_kernel<KV, D, R>, smem);
    if (e != cudaSuccess) return e;
    const Plan p = make_plan(KV, a.Hq / a.kv.n_kv, a.kv.n_kv, a.B, a.kv.max_pages, sm_count);
    e = launch_dependent(decode_attn_kernel<KV, D, R>, dim3(p.blocks), kThreads, smem, 1, s, a, p);
    if (e != cudaSuccess || most_units(KV, a.kv.max_pages) <= L::kJoinUnits) return e;  // no item of this table is ever cut
    using Act = typename std::conditional<KV == VELO_KV_F32, float, __half>::type;
    // Few items are cut into many states each: 4 warps per query head.  Otherwise most blocks have
    // nothing to join and only have to leave soon: one of 8 warps for (8 of) an item's heads.
    constexpr int rows = rows_of(R), each = rows < 8 ? rows : 8;
    if ((long long)a.B * a.kv.n_kv * p.tiles <= 16)
        return launch_dependent(decode_join_kernel<Act, D, 4, 1>, dim3(p.blocks, rows), 128, 0, 1, s, a, p, rows);
    return launch_dependent(decode_join_kernel<Act, D, 8, each>, dim3(p.blocks, rows / each), 256, 0, 1, s, a, p, rows);
}

template <int KV, int R>
cudaError_t launch_rows(const DecodeAttnArgs& a, int sm_count, cudaStream_t s) {
    return a.kv.head_dim == 64 ? launch_typed<KV, 64, R>(a, sm_count, s) : launch_typed<KV, 128, R>(a, sm_count, s);
}

}  // namespace

int64_t decode_attn_steps(int Hq, int Hkv, int kv_dtype, int max_pages) {
    const int group = Hq / Hkv, rows = rows_of(row_tiles(group, kv_dtype));
    return (int64_t)Hkv * ((group + rows - 1) / rows) * most_units(kv_dtype, max_pages);
}

size_t decode_attn_workspace(int Hq, int Hkv, int D, int sm_count) {
    // the most that any page type needs
    size_t most = 0;
    for (int kv : {VELO_KV_F16, VELO_KV_INT8, VELO_KV_F32}) {
        const int R = row_tiles(Hq / Hkv, kv);
        const size_t blocks = all_blocks(kv, R, sm_count);
        most = std::max(most, blocks * (sizeof(int4) + 2 * slot_floats(rows_of(R), D) * sizeof(float)));
    }
    return most;
}

cudaError_t launch_decode_attention(const DecodeAttnArgs& a, int sm_count, cudaStream_t s) {
    const int R = row_tiles(a.Hq / a.kv.n_kv, a.kv.kv_dtype);
    if (a.kv.kv_dtype == VELO_KV_F32) return launch_rows<VELO_KV_F32, 1>(a, sm_count, s);
    if (a.kv.kv_dtype == VELO_KV_INT8)
        return R == 2   ? launch_rows<VELO_KV_INT8, 2>(a, sm_count, s)
               : R == 1 ? launch_rows<VELO_KV_INT8, 1>(a, sm_count, s)
                        : launch_rows<VELO_KV_INT8, 0>(a, sm_count, s);
    return R == 2   ? launch_rows<VELO_KV_F16, 2>(a, sm_count, s)
           : R == 1 ? launch_rows<VELO_KV_F16, 1>(a, sm_count, s)
                    : launch_rows<VELO_KV_F16, 0>(a, sm_count, s);
}

}  // namespace velo
