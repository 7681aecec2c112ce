// paged_append.cu -- new tokens into a paged key-value cache: per-head
// RMSNorm, rotary embedding and rounding to the cache's 16-bit type, queries
// to a buffer, keys and values to the pages (abra_paged_append).
//
// For a head x of D values with norm weights w and the table row (c_i, s_i) of
// the token's position: y = x * rsqrt(mean(x^2) + eps) * w, then for i < D/2
//   o_i = y_i c_i - y_{i+D/2} s_i,   o_{i+D/2} = y_{i+D/2} c_i + y_i s_i.
// Everything is fp32 up to the one rounding of the store.
#include "paged_kv.cuh"

namespace abra {
namespace {

struct AppendArgs {
    PagedKv kv;
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv, ldqo;
    const int32_t *cu_new;
    const float *q_norm, *k_norm, *rope;
    void *q_out;
    float eps;
    int n_heads, n_tokens, rope_len;
};

// Sequence of token t: the last s with cu_new[s] <= t.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int n_seqs, int t) {
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= t) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__half x) { return __half2float(x); }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }

constexpr int APPEND_WARPS = 8;

// One warp per (token, head).  Lane l holds the pairs (i, i + D/2) for i = l,
// l + 32.
template <typename TI, typename T, int D>
__global__ void __launch_bounds__(APPEND_WARPS * 32) append_kernel(const __grid_constant__ AppendArgs p) {
    constexpr int HALF = D / 2, NP = (HALF + 31) / 32;
    const int lane = threadIdx.x & 31;
    const int heads = (p.q ? p.n_heads : 0) + 2 * p.kv.a.n_kv_heads;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * APPEND_WARPS + (threadIdx.x >> 5);
    if (item >= static_cast<int64_t>(p.n_tokens) * heads) return;
    const int t = static_cast<int>(item / heads);
    int h = static_cast<int>(item - static_cast<int64_t>(t) * heads);
    int kind = 0;  // 0 query, 1 key, 2 value
    if (!p.q) kind = 1;
    else if (h >= p.n_heads) { kind = 1; h -= p.n_heads; }
    if (kind && h >= p.kv.a.n_kv_heads) { kind = 2; h -= p.kv.a.n_kv_heads; }
    // the token's sequence, slot and position
    int s, end;
    if (p.cu_new) {
        s = sequence_of(p.cu_new, p.kv.a.n_seqs, t);
        end = __ldg(p.cu_new + s + 1);
    } else {
        const int m = p.n_tokens / p.kv.a.n_seqs;
        s = t / m;
        end = (s + 1) * m;
    }
    const int len = paged_len(p.kv, s);
    const int slot = len - (end - t), at = paged_next_pos(p.kv, s, len) - (end - t);

    const TI *src = static_cast<const TI *>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                    t * (kind == 0 ? p.ldq : kind == 1 ? p.ldk : p.ldv) + static_cast<int64_t>(h) * D;
    float lo[NP], hi[NP];
#pragma unroll
    for (int u = 0; u < NP; ++u) {
        const int i = lane + 32 * u;
        lo[u] = i < HALF ? up(src[i]) : 0.0f;
        hi[u] = i < HALF ? up(src[i + HALF]) : 0.0f;
    }
    const float *nw = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
    if (nw) {
        float ss = 0.0f;
#pragma unroll
        for (int u = 0; u < NP; ++u) ss += lo[u] * lo[u] + hi[u] * hi[u];
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float r = rsqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int i = lane + 32 * u;
            if (i < HALF) {
                lo[u] *= r * __ldg(nw + i);
                hi[u] *= r * __ldg(nw + i + HALF);
            }
        }
    }
    if (p.rope && kind < 2) {
        if (at >= 0 && at < p.rope_len) {
            const float2 *row = reinterpret_cast<const float2 *>(p.rope) + static_cast<int64_t>(at) * HALF;
#pragma unroll
            for (int u = 0; u < NP; ++u) {
                const int i = lane + 32 * u;
                if (i < HALF) {
                    const float2 cs = __ldg(row + i);
                    const float a = lo[u], b = hi[u];
                    lo[u] = a * cs.x - b * cs.y;
                    hi[u] = b * cs.x + a * cs.y;
                }
            }
        } else if (lane == 0) {
            report_error(ERR_BAD_INDEX);
        }
    }
    T *dst;
    if (kind == 0) {
        dst = static_cast<T *>(p.q_out) + t * p.ldqo + static_cast<int64_t>(h) * D;
    } else {
        if (slot < 0) {  // more new tokens than the sequence has slots
            if (lane == 0) report_error(ERR_BAD_INDEX);
            return;
        }
        const int e = p.kv.page.div(slot), off = slot - e * p.kv.a.page_size;
        const int page = paged_page(p.kv, s, e);
        if (page < 0) return;
        dst = kind == 1 ? static_cast<T *>(p.kv.a.k) + paged_k_at(p.kv, page, h, off)
                        : static_cast<T *>(p.kv.a.v) + paged_v_at(p.kv, page, h, off);
        if (kind == 1 && lane == 0) {
            const int64_t m = paged_meta_at(p.kv, page, h, off);
            if (p.kv.a.acc) p.kv.a.acc[m] = 0.0f;
            if (p.kv.a.pos) p.kv.a.pos[m] = at;
        }
    }
#pragma unroll
    for (int u = 0; u < NP; ++u) {
        const int i = lane + 32 * u;
        if (i < HALF) {
            dst[i] = Half16<T>::down(lo[u]);
            dst[i + HALF] = Half16<T>::down(hi[u]);
        }
    }
}

template <typename TI, typename T>
cudaError_t launch(const AppendArgs &p, cudaStream_t stream) {
    const int64_t heads = (p.q ? p.n_heads : 0) + 2 * p.kv.a.n_kv_heads;
    const int64_t items = p.n_tokens * heads;
    const dim3 grid(static_cast<unsigned>((items + APPEND_WARPS - 1) / APPEND_WARPS));
    switch (p.kv.a.head_dim) {
        case 64: append_kernel<TI, T, 64><<<grid, APPEND_WARPS * 32, 0, stream>>>(p); break;
        case 96: append_kernel<TI, T, 96><<<grid, APPEND_WARPS * 32, 0, stream>>>(p); break;
        default: append_kernel<TI, T, 128><<<grid, APPEND_WARPS * 32, 0, stream>>>(p); break;
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace abra

ABRA_ERROR_WORD_ACCESSOR(paged_append_error_word)

extern "C" int abra_paged_append(const abra_paged_kv *kv, const void *q, const void *k, const void *v,
                                 int32_t in_type, int64_t ldq, int64_t ldk, int64_t ldv,
                                 int32_t n_heads, const int32_t *cu_new, int32_t n_tokens,
                                 const float *q_norm, const float *k_norm, float eps,
                                 const float *rope, int32_t rope_len, void *q_out, int64_t ldqo,
                                 void *stream) {
    using namespace abra;
    int rc = paged_check(kv);
    if (rc) return rc;
    if (in_type != ABRA_GGML_F32 && in_type != ABRA_GGML_F16 && in_type != ABRA_GGML_BF16)
        return paged_fail(ABRA_E_UNSUPPORTED, "the tokens' type must be F32, F16 or BF16 (got %d)", in_type);
    if (n_tokens < 0) return paged_fail(ABRA_E_INVALID, "n_tokens must not be negative");
    if (!cu_new && kv->n_seqs > 0 && n_tokens % kv->n_seqs)
        return paged_fail(ABRA_E_INVALID, "without cu_new n_tokens (%d) must be a multiple of n_seqs (%d)", n_tokens,
                          kv->n_seqs);
    if (kv->n_seqs == 0 && n_tokens > 0) return paged_fail(ABRA_E_INVALID, "tokens without a sequence");
    if (n_tokens == 0) return ABRA_OK;
    if (!k || !v || (q != nullptr) != (q_out != nullptr))
        return paged_fail(ABRA_E_INVALID, "null k or v, or only one of q and q_out");
    if (q && n_heads < 1) return paged_fail(ABRA_E_INVALID, "n_heads must be positive");
    if (n_heads > 65535) return paged_fail(ABRA_E_UNSUPPORTED, "over 65535 heads");
    const int64_t kvw = static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim;
    const int64_t qw = static_cast<int64_t>(n_heads) * kv->head_dim;
    if (ldk < kvw || ldv < kvw || (q && (ldq < qw || ldqo < qw)))
        return paged_fail(ABRA_E_INVALID, "a row stride is smaller than its heads");
    const int64_t lds = ldk | ldv | (q ? ldq | ldqo : 0);
    if (lds % 8 || !paged_aligned(k, 16) || !paged_aligned(v, 16) || !paged_aligned(q, 16) || !paged_aligned(q_out, 16))
        return paged_fail(ABRA_E_INVALID, "rows must start on 16 bytes and their strides be multiples of 8 elements");
    if (!paged_aligned(q_norm, 16) || !paged_aligned(k_norm, 16) || !paged_aligned(rope, 16) || !paged_aligned(cu_new, 4))
        return paged_fail(ABRA_E_INVALID, "norm weights and rope must be 16-byte aligned");
    if (rope && rope_len < 1) return paged_fail(ABRA_E_INVALID, "rope_len must be positive");
    const int64_t heads = (q ? n_heads : 0) + 2ll * kv->n_kv_heads;
    if (n_tokens * heads > (1ll << 33)) return paged_fail(ABRA_E_UNSUPPORTED, "n_tokens * heads over 2^33");
    AppendArgs p{paged_view(kv), q, k, v, ldq, ldk, ldv, ldqo, cu_new, q_norm, k_norm, rope, q_out, eps, n_heads, n_tokens, rope_len};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (kv->type == ABRA_GGML_F16)
        e = in_type == ABRA_GGML_F32   ? launch<float, __half>(p, st)
            : in_type == ABRA_GGML_F16 ? launch<__half, __half>(p, st)
                                       : launch<__nv_bfloat16, __half>(p, st);
    else
        e = in_type == ABRA_GGML_F32   ? launch<float, __nv_bfloat16>(p, st)
            : in_type == ABRA_GGML_F16 ? launch<__half, __nv_bfloat16>(p, st)
                                       : launch<__nv_bfloat16, __nv_bfloat16>(p, st);
    return paged_cuda(e, "paged append launch");
}
