// decode.cu -- C ABI of one-token decoding over a caller's paged cache
// (include/velo_cuda.h): kv_append, decode_attention, token_logprobs.
#include <cmath>

#include "kernels/decode_ops.h"
#include "runtime/context.h"

using velo::fail;

namespace {

// Makes the context's device current for a scope and restores the caller's.
struct DeviceScope {
    int before = -1;
    cudaError_t st;
    explicit DeviceScope(int device) {
        st = cudaGetDevice(&before);
        if (st == cudaSuccess && before != device)
            st = cudaSetDevice(device);
        else
            before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

bool misaligned(const void* p, size_t a = 16) { return (uintptr_t)p % a != 0; }

int elem_bytes(int32_t dtype) { return dtype == VELO_ELEM_F32 ? 4 : 2; }

constexpr int kMaxHeads = 1 << 16;  // products of heads, tokens and pages then stay in 64 bits

bool bad_heads(int32_t n_head, int32_t n_kv) {
    return n_kv < 1 || n_head < n_kv || n_head > kMaxHeads || n_head % n_kv;
}

int32_t check_cache(const char* op, const velo_kv_cache* k, velo::PagedKv& out) {
    if (!k) return fail(VELO_ERR_INVALID_ARGUMENT, "%s: cache is NULL", op);
    if (k->struct_size != sizeof(velo_kv_cache))
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: velo_kv_cache.struct_size %u != %zu", op, k->struct_size,
                    sizeof(velo_kv_cache));
    if (k->kv_dtype < VELO_KV_F16 || k->kv_dtype > VELO_KV_F32)
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: kv_dtype %d", op, k->kv_dtype);
    if (k->head_dim != 64 && k->head_dim != 128)
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: head_dim %d unsupported (64 or 128)", op, k->head_dim);
    if (k->n_kv < 1 || k->n_kv > kMaxHeads || k->pool_pages < 1 || k->max_pages < 0 || k->max_pages > 1 << 26)
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: n_kv %d, pool_pages %d, max_pages %d", op, k->n_kv,
                    k->pool_pages, k->max_pages);
    if (!k->k_pool || !k->v_pool || (k->max_pages > 0 && !k->page_table) ||
        (k->kv_dtype == VELO_KV_INT8 && (!k->k_scale || !k->v_scale)))
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: NULL pool, scale or page table", op);
    if (misaligned(k->k_pool) || misaligned(k->v_pool) || misaligned(k->page_table, 4) ||
        (k->kv_dtype == VELO_KV_INT8 && (misaligned(k->k_scale) || misaligned(k->v_scale))))
        return fail(VELO_ERR_INVALID_ARGUMENT, "%s: pools and scales must be 16-byte aligned", op);
    out.k_pool = k->k_pool;
    out.v_pool = k->v_pool;
    out.k_scale = static_cast<__half*>(k->k_scale);
    out.v_scale = static_cast<__half*>(k->v_scale);
    out.page_table = k->page_table;
    out.pool_pages = k->pool_pages;
    out.max_pages = k->max_pages;
    out.n_kv = k->n_kv;
    out.head_dim = k->head_dim;
    out.kv_dtype = k->kv_dtype;
    return VELO_OK;
}

// The rotation table of (base, head_dim); the context keeps the last one.
const velo::RopeTurns& rope_turns(velo_cuda_ctx* c, float base, int D) {
    if (c->rope_base != base || c->rope_dim != D) {
        // (the extended type's 64-bit mantissa: a double would leave 2^-56 turns per position)
        const long double two_pi = 6.283185307179586476925286766559L;
        for (int i = 0; i < D / 2; ++i)
            c->rope_turns[i] =
                (uint64_t)std::floor(std::ldexp(std::pow((long double)base, -2.0L * i / D) / two_pi, 64) + 0.5L);
        c->rope_base = base;
        c->rope_dim = D;
    }
    return *reinterpret_cast<const velo::RopeTurns*>(c->rope_turns);
}

}  // namespace

extern "C" {

int32_t velo_cuda_kv_append(velo_cuda_ctx* c, const velo_kv_cache* cache, const velo_kv_append_batch* in) {
    velo::Range nvtx_range("velo.kv_append");
    velo::clear_last_error();
    if (!c) return fail(VELO_ERR_INVALID_ARGUMENT, "ctx is NULL");
    velo::KvAppendArgs a{};
    int32_t st = check_cache("kv_append", cache, a.kv);
    if (st) return st;
    if (!in) return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: batch is NULL");
    if (in->struct_size != sizeof(velo_kv_append_batch))
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: velo_kv_append_batch.struct_size %u != %zu", in->struct_size,
                    sizeof(velo_kv_append_batch));
    const int D = cache->head_dim, n_kv = cache->n_kv;
    if (in->in_dtype < VELO_ELEM_F32 || in->in_dtype > VELO_ELEM_BF16)
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: in_dtype %d", in->in_dtype);
    if (in->n_head != 0 && bad_heads(in->n_head, n_kv))
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: n_head %d / n_kv %d", in->n_head, n_kv);
    if (!(in->freq_base > 1.0f) || std::isinf(in->freq_base))
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: freq_base must be finite and above 1");
    if (in->B < 0 || in->n_tokens < 0 || (!in->seq_start && in->n_tokens != in->B))
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: B %d, n_tokens %d%s", in->B, in->n_tokens,
                    in->seq_start ? "" : " without seq_start");
    if ((int64_t)in->n_tokens * (in->n_head + 2 * (int64_t)n_kv) >= (int64_t)1 << 31)
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: %d tokens of %d heads are too many", in->n_tokens, in->n_head);
    if (in->B == 0 || in->n_tokens == 0) return VELO_OK;
    if (!in->k || !in->v || !in->ctx_len || !in->q != !in->q_out || !in->q != (in->n_head == 0) || !in->k_out != !in->v_out)
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: NULL buffer");
    const int eb = elem_bytes(in->in_dtype);
    if ((in->q && (misaligned(in->q) || misaligned(in->q_out) || in->ldq * eb % 16)) || misaligned(in->k) ||
        misaligned(in->v) || in->ldk * eb % 16 || in->ldv * eb % 16 || misaligned(in->k_out) || misaligned(in->v_out) ||
        misaligned(in->seq_start, 4) || misaligned(in->ctx_len, 4))
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: rows must be 16-byte aligned");
    if ((in->q && in->ldq < (int64_t)in->n_head * D) || in->ldk < (int64_t)n_kv * D || in->ldv < (int64_t)n_kv * D)
        return fail(VELO_ERR_INVALID_ARGUMENT, "kv_append: row stride below the row (ldq %lld, ldk %lld, ldv %lld)",
                    (long long)in->ldq, (long long)in->ldk, (long long)in->ldv);
    DeviceScope dev(c->device);
    VELO_CUDA_TRY(dev.st);
    a.q = in->q;
    a.k = in->k;
    a.v = in->v;
    a.in_dtype = in->in_dtype;
    a.ldq = in->ldq;
    a.ldk = in->ldk;
    a.ldv = in->ldv;
    a.seq_start = in->seq_start;
    a.ctx_len = in->ctx_len;
    a.B = in->B;
    a.T = in->n_tokens;
    a.Hq = in->n_head;
    a.q_out = in->q_out;
    a.k_out = in->k_out;
    a.v_out = in->v_out;
    a.err = c->err_flag;
    a.turns = rope_turns(c, in->freq_base, D);
    VELO_CUDA_TRY(velo::launch_kv_append(a, c->stream));
    return VELO_OK;
}

size_t velo_cuda_decode_attention_workspace(velo_cuda_ctx* c, int32_t n_head, int32_t n_kv, int32_t head_dim) {
    if (!c || bad_heads(n_head, n_kv) || (head_dim != 64 && head_dim != 128)) return 0;
    return velo::decode_attn_workspace(n_head, n_kv, head_dim, c->sm_count);
}

int32_t velo_cuda_decode_attention(velo_cuda_ctx* c, const velo_kv_cache* cache, const void* q, int64_t ldq,
                                   const int32_t* seq_len, int32_t B, int32_t n_head, float scale, void* out,
                                   float* lse, void* workspace, size_t workspace_bytes) {
    velo::Range nvtx_range("velo.decode_attention");
    velo::clear_last_error();
    if (!c) return fail(VELO_ERR_INVALID_ARGUMENT, "ctx is NULL");
    velo::DecodeAttnArgs a{};
    int32_t st = check_cache("decode_attention", cache, a.kv);
    if (st) return st;
    if (bad_heads(n_head, cache->n_kv))
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: n_head %d / n_kv %d", n_head, cache->n_kv);
    if (B < 0 || B > velo::kDecodeMaxB)
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: B %d outside [0, %d]", B, velo::kDecodeMaxB);
    if (!(scale >= 0.0f) || std::isinf(scale))
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: scale must be finite and >= 0");
    const int64_t steps = B * velo::decode_attn_steps(n_head, cache->n_kv, cache->kv_dtype, cache->max_pages);
    if (steps > velo::kDecodeMaxSteps)
        return fail(VELO_ERR_INVALID_ARGUMENT,
                    "decode_attention: %d page-table rows of %d pages are %lld steps of work, above 2^30", B,
                    cache->max_pages, (long long)steps);
    if (B == 0) return VELO_OK;
    if (!q || !seq_len || !out) return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: NULL buffer");
    const int eb = cache->kv_dtype == VELO_KV_F32 ? 4 : 2;
    if (misaligned(q) || misaligned(out) || ldq * eb % 16 || misaligned(seq_len, 4) || misaligned(lse, 4))
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: rows must be 16-byte aligned");
    if (ldq < (int64_t)n_head * cache->head_dim)
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: ldq %lld below the row", (long long)ldq);
    const size_t need = velo::decode_attn_workspace(n_head, cache->n_kv, cache->head_dim, c->sm_count);
    if (need && (!workspace || misaligned(workspace) || workspace_bytes < need))
        return fail(VELO_ERR_INVALID_ARGUMENT, "decode_attention: workspace of %zu bytes, 16-byte aligned, needed",
                    need);
    DeviceScope dev(c->device);
    VELO_CUDA_TRY(dev.st);
    a.q = q;
    a.ldq = ldq;
    a.seq_len = seq_len;
    a.B = B;
    a.Hq = n_head;
    a.scale = scale > 0.0f ? scale : (float)(1.0 / std::sqrt((double)cache->head_dim));
    a.out = out;
    a.lse = lse;
    a.ws = workspace;
    a.err = c->err_flag;
    VELO_CUDA_TRY(velo::launch_decode_attention(a, c->sm_count, c->stream));
    return VELO_OK;
}

int32_t velo_cuda_token_logprobs(velo_cuda_ctx* c, const void* logits, int32_t logits_dtype, int64_t ldl, int32_t M,
                                 int32_t V, const uint32_t* tokens, float temperature, float* logprob,
                                 float* entropy, int32_t n_top, uint32_t* top_tokens, float* top_logprobs) {
    velo::Range nvtx_range("velo.token_logprobs");
    velo::clear_last_error();
    if (!c) return fail(VELO_ERR_INVALID_ARGUMENT, "ctx is NULL");
    if (logits_dtype < VELO_ELEM_F32 || logits_dtype > VELO_ELEM_BF16)
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: logits_dtype %d", logits_dtype);
    if (M < 0 || V < 1 || V > 1 << 24)
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: M = %d, V = %d outside [1, 2^24]", M, V);
    if (n_top < 0 || n_top > velo::kMaxTop || n_top > V)
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: n_top = %d outside [0, min(%d, V)]", n_top,
                    velo::kMaxTop);
    if (!(temperature >= 1e-30f && temperature <= 1e30f))
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: temperature outside [1e-30, 1e30]");
    if (ldl < V) return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: ldl %lld < V = %d", (long long)ldl, V);
    if (M == 0) return VELO_OK;
    if (!logits || !tokens != !logprob || (n_top > 0 && (!top_tokens || !top_logprobs)))
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: NULL buffer");
    if (misaligned(logits, elem_bytes(logits_dtype)) || misaligned(tokens, 4) || misaligned(logprob, 4) ||
        misaligned(entropy, 4) || misaligned(top_tokens, 4) || misaligned(top_logprobs, 4))
        return fail(VELO_ERR_INVALID_ARGUMENT, "token_logprobs: misaligned buffer");
    if (!logprob && !entropy && n_top == 0) return VELO_OK;
    DeviceScope dev(c->device);
    VELO_CUDA_TRY(dev.st);
    velo::TokenLogprobsArgs a{};
    a.logits = logits;
    a.dtype = logits_dtype;
    a.ldl = ldl;
    a.M = M;
    a.V = V;
    a.tokens = tokens;
    a.inv_t = 1.0f / temperature;
    a.logprob = logprob;
    a.entropy = entropy;
    a.n_top = n_top;
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    a.err = c->err_flag;
    VELO_CUDA_TRY(velo::launch_token_logprobs(a, c->sm_count, c->stream));
    return VELO_OK;
}

}  // extern "C"
