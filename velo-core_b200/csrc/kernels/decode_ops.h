// decode_ops.h -- kernels of one-token decoding over a caller's paged cache:
// K/V append with rotation (kv_append.cu), decode attention (decode_attn.cu)
// and token log probabilities (token_logprobs.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace velo {

constexpr int kPageTokens = 16;

// The caller's cache, as velo_kv_cache describes it.
struct PagedKv {
    void* k_pool;
    void* v_pool;
    __half* k_scale;
    __half* v_scale;
    const uint32_t* page_table;
    int pool_pages, max_pages, n_kv, head_dim, kv_dtype;
};

// base^(-2i/D) / 2pi of every rotation pair, in turns: 64-bit binary fractions,
// so that position x frequency modulo one turn is one wrapping multiplication,
// off by no more than 2^-64 turns per position.
struct RopeTurns {
    uint64_t f[64];
};

struct KvAppendArgs {
    PagedKv kv;
    const void* q;
    const void* k;
    const void* v;
    int in_dtype;  // velo_elem
    long long ldq, ldk, ldv;
    const int32_t* seq_start;
    const int32_t* ctx_len;
    int B, T, Hq;
    void* q_out;
    void* k_out;
    void* v_out;
    int* err;
    RopeTurns turns;
};
cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s);

constexpr int kDecodeMaxB = 4096;
struct DecodeAttnArgs {
    PagedKv kv;
    const void* q;
    long long ldq;
    const int32_t* seq_len;
    int B, Hq;
    float scale;
    void* out;
    float* lse;
    void* ws;
    int* err;
};
// Steps of work that one sequence filling its page-table row makes; the list of a call
// is counted in 32 bits.
constexpr int64_t kDecodeMaxSteps = (int64_t)1 << 30;
int64_t decode_attn_steps(int Hq, int Hkv, int kv_dtype, int max_pages);
size_t decode_attn_workspace(int Hq, int Hkv, int D, int sm_count);
cudaError_t launch_decode_attention(const DecodeAttnArgs& a, int sm_count, cudaStream_t s);

constexpr int kMaxTop = 64;
struct TokenLogprobsArgs {
    const void* logits;
    int dtype;  // velo_elem
    long long ldl;
    int M, V;
    const uint32_t* tokens;
    float inv_t;
    float* logprob;
    float* entropy;
    int n_top;
    uint32_t* top_tokens;
    float* top_logprobs;
    int* err;
};
cudaError_t launch_token_logprobs(const TokenLogprobsArgs& a, int sm_count, cudaStream_t s);

}  // namespace velo
