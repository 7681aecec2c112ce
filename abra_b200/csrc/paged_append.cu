// paged_append.cu -- new tokens into a paged key-value cache: per-head
// RMSNorm, rotary embedding and rounding to the cache's 16-bit type, queries
// to a buffer, keys and values to the pages (abra_paged_append).
//
// For a head x of D values with norm weights w and the table row (c_i, s_i) of
// the token's position: y = x * rsqrt(mean(x^2) + eps) * w, then for i < D/2
//   o_i = y_i c_i - y_{i+D/2} s_i,   o_{i+D/2} = y_{i+D/2} c_i + y_i s_i.
// Everything is fp32 up to the one rounding of the store.
//
// Bound: 4 bytes read and 2 written a value; for few tokens the way from the
// launch through the token's lookups to the store.  Measured (B200, 1965 MHz, 32
// + 8 + 8 heads of 128): 9,555 tokens of prompts, 358 MB, 64 us = 5.6 TB/s, with
// 61 % of the issue slots used; one token 4.5 us, 32 of as many sequences 4.7.  From
// 16-bit tokens 84 us: they are converted where they are loaded, so that these loads
// do not run ahead (5.5 warps a scheduler wait for them, 1.7 with fp32).
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
    int tokens;     // of a CTA
    FastDiv heads;  // heads of a token, queries, keys and values
};

// Four neighbouring values.
__device__ __forceinline__ float4 load4(const float *p) { return __ldcs(reinterpret_cast<const float4 *>(p)); }
template <typename T> __device__ __forceinline__ float4 load4(const T *p) {
    const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(p));
    const T *h = reinterpret_cast<const T *>(&x);
    return make_float4(Half16<T>::up(h[0]), Half16<T>::up(h[1]), Half16<T>::up(h[2]), Half16<T>::up(h[3]));
}
template <typename T> __device__ __forceinline__ void store4(T *p, float4 x) {
    const T h[4] = {Half16<T>::down(x.x), Half16<T>::down(x.y), Half16<T>::down(x.z), Half16<T>::down(x.w)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(h);
}
__device__ __forceinline__ float4 read4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 mul4(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_TOKENS = 4;  // of a CTA, where there are many (2: 67 us, 8: 71, for 64 us)

// A CTA takes a few neighbouring tokens, a group of 16 lanes (8 for heads of
// 64) a head: lane j holds the pairs (4 j + u, 4 j + u + D/2), u = 0..3.  The
// first heads' values are asked for before the tokens' sequences, slots and
// pages are looked up, so that the chain of small reads (offsets, length,
// table) runs under the large ones, and several tokens share it; after that the
// next heads' loads run under this batch's arithmetic and stores (69 us without).
template <typename TI, typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS, 4) append_kernel(const __grid_constant__ AppendArgs p) {
    constexpr int HALF = D / 2, LANES = D == 64 ? 8 : 16, GROUPS = APPEND_THREADS / LANES, BATCH = 2;
    __shared__ int s_page[APPEND_TOKENS], s_off[APPEND_TOKENS], s_at[APPEND_TOKENS];
    pdl_wait();
    pdl_launch_dependents();
    const int group = threadIdx.x / LANES, j = threadIdx.x % LANES;
    const unsigned lanes = ((1u << LANES) - 1u) << (threadIdx.x % 32 / LANES * LANES);  // the group's
    const bool on = 4 * j < HALF;  // heads of 96 use 12 lanes of a group
    const int nq = p.q ? p.n_heads : 0, nkv = p.kv.a.n_kv_heads, heads = nq + 2 * nkv;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.n_tokens - t0)), items = nt * heads;
    float4 lo[BATCH], hi[BATCH], lo_next[BATCH], hi_next[BATCH];
    auto load = [&](int base, float4 (&lo)[BATCH], float4 (&hi)[BATCH]) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int x = base + b * GROUPS;
            lo[b] = hi[b] = make_float4(0, 0, 0, 0);
            if (x >= items || !on) continue;
            const int i = p.heads.div(x), h = x - i * heads;
            const int64_t t = t0 + i;
            const TI *src = h < nq         ? static_cast<const TI *>(p.q) + t * p.ldq + static_cast<int64_t>(h) * D
                            : h < nq + nkv ? static_cast<const TI *>(p.k) + t * p.ldk + static_cast<int64_t>(h - nq) * D
                                           : static_cast<const TI *>(p.v) + t * p.ldv + static_cast<int64_t>(h - nq - nkv) * D;
            lo[b] = load4(src + 4 * j);
            hi[b] = load4(src + 4 * j + HALF);
        }
    };
    int base = group;
    load(base, lo, hi);
    // the first token's sequence: how many end at or before it
    int s = 0;
    if (p.cu_new) {
        for (int x = 0; x < p.kv.a.n_seqs; x += APPEND_THREADS) {
            const int y = x + threadIdx.x;
            const int ends = y < p.kv.a.n_seqs ? p.cu_new[y + 1] : 0x7fffffff;
            s += __syncthreads_count(ends <= t0);
            // one CTA looks at all offsets' order and ends
            if (blockIdx.x == 0 && y < p.kv.a.n_seqs) {
                const int starts = p.cu_new[y];
                if (starts > ends || (y == 0 && starts != 0) || (y == p.kv.a.n_seqs - 1 && ends != p.n_tokens)) report_error(ERR_BAD_INDEX);
            }
        }
    }
    if (threadIdx.x < nt) {  // each token's slot, position and page
        const int t = static_cast<int>(t0) + threadIdx.x;
        int end, page = -1, off = 0, at = -1;
        bool mine;  // the offsets give the token to sequence s
        if (p.cu_new) {
            while (s < p.kv.a.n_seqs && p.cu_new[s + 1] <= t) ++s;
            end = s < p.kv.a.n_seqs ? p.cu_new[s + 1] : 0;
            mine = s < p.kv.a.n_seqs && p.cu_new[s] <= t && end <= p.n_tokens;
        } else {
            const int m = p.n_tokens / p.kv.a.n_seqs;
            s = t / m;
            end = (s + 1) * m;
            mine = true;
        }
        if (mine) {
            const int len = paged_len(p.kv, s), slot = len - (end - t);
            at = paged_next_pos(p.kv, s, len) - (end - t);
            if (slot >= 0) {
                const int e = p.kv.page.div(slot);
                off = slot - e * p.kv.a.page_size;
                page = paged_page(p.kv, s, e);
            }
            if (slot < 0 || (p.rope && (at < 0 || at >= p.rope_len))) report_error(ERR_BAD_INDEX);
        } else {
            report_error(ERR_BAD_INDEX);
        }
        s_page[threadIdx.x] = page, s_off[threadIdx.x] = off, s_at[threadIdx.x] = at;
    }
    __syncthreads();
    for (;;) {
        load(base + BATCH * GROUPS, lo_next, hi_next);  // zeros beyond the last item
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int item = base + b * GROUPS;
            if (item >= items) break;  // the whole group
            const int i = p.heads.div(item), h = item - i * heads, page = s_page[i], at = s_at[i];
            float4 x = lo[b], y = hi[b];
            const float *nw = h < nq ? p.q_norm : h < nq + nkv ? p.k_norm : nullptr;
            if (nw) {
                float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + (y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w);
#pragma unroll
                for (int m = LANES / 2; m >= 1; m >>= 1) ss += __shfl_xor_sync(lanes, ss, m);
                const float r = rsqrtf(ss * (1.0f / D) + p.eps);
                if (on) {
                    x = mul4(mul4(x, make_float4(r, r, r, r)), read4(nw + 4 * j));
                    y = mul4(mul4(y, make_float4(r, r, r, r)), read4(nw + 4 * j + HALF));
                }
            }
            if (p.rope && h < nq + nkv && on && at >= 0 && at < p.rope_len) {
                const float *row = p.rope + static_cast<int64_t>(at) * D + 8 * j;
                const float4 c01 = read4(row), c23 = read4(row + 4), u = x;  // cos, sin of two pairs each
                x = make_float4(u.x * c01.x - y.x * c01.y, u.y * c01.z - y.y * c01.w, u.z * c23.x - y.z * c23.y,
                                u.w * c23.z - y.w * c23.w);
                y = make_float4(y.x * c01.x + u.x * c01.y, y.y * c01.z + u.y * c01.w, y.z * c23.x + u.z * c23.y,
                                y.w * c23.z + u.w * c23.w);
            }
            T *dst = nullptr;
            if (h < nq) {
                dst = static_cast<T *>(p.q_out) + (t0 + i) * p.ldqo + static_cast<int64_t>(h) * D;
            } else if (page >= 0) {
                if (h < nq + nkv) {
                    dst = static_cast<T *>(p.kv.a.k) + paged_k_at(p.kv, page, h - nq, s_off[i]);
                    if (j == 0) {
                        const int64_t m = paged_meta_at(p.kv, page, h - nq, s_off[i]);
                        if (p.kv.a.acc) p.kv.a.acc[m] = 0.0f;
                        if (p.kv.a.pos) p.kv.a.pos[m] = at;
                    }
                } else {
                    dst = static_cast<T *>(p.kv.a.v) + paged_v_at(p.kv, page, h - nq - nkv, s_off[i]);
                }
            }
            if (dst && on) {
                store4(dst + 4 * j, x);
                store4(dst + 4 * j + HALF, y);
            }
        }
        base += BATCH * GROUPS;
        if (base >= items) return;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) lo[b] = lo_next[b], hi[b] = hi_next[b];
    }
}

template <typename TI, typename T>
cudaError_t launch(const AppendArgs &p, cudaStream_t stream) {
    const dim3 grid((p.n_tokens - 1) / p.tokens + 1);
    switch (p.kv.a.head_dim) {
        case 64: return paged_launch(append_kernel<TI, T, 64>, grid, APPEND_THREADS, 0, stream, p);
        case 96: return paged_launch(append_kernel<TI, T, 96>, grid, APPEND_THREADS, 0, stream, p);
        default: return paged_launch(append_kernel<TI, T, 128>, grid, APPEND_THREADS, 0, stream, p);
    }
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
    const int64_t kvw = static_cast<int64_t>(kv->n_kv_heads) * kv->head_dim;
    const int64_t qw = static_cast<int64_t>(n_heads) * kv->head_dim;
    if (ldk < kvw || ldv < kvw || (q && (ldq < qw || ldqo < qw)))
        return paged_fail(ABRA_E_INVALID, "a row stride is smaller than its heads");
    const int64_t lds = ldk | ldv | (q ? ldq | ldqo : 0);
    if (lds % 8 || !paged_aligned(k, 16) || !paged_aligned(v, 16) || !paged_aligned(q, 16) || !paged_aligned(q_out, 16))
        return paged_fail(ABRA_E_INVALID, "rows must start on 16 bytes and their strides be multiples of 8 elements");
    if (!paged_aligned(q_norm, 16) || !paged_aligned(k_norm, 16) || !paged_aligned(rope, 16) || !paged_aligned(cu_new, 4))
        return paged_fail(ABRA_E_INVALID, "norm weights and rope must be 16-byte aligned");
    if (q) {
        // heads are stored while others are still to be read; a head of 16-bit values may take its own place
        const int64_t in = in_type == ABRA_GGML_F32 ? 4 : 2;
        const PagedRows to{q_out, 2 * qw, 2 * ldqo};
        const bool own = q == q_out && in == 2 && ldq == ldqo;
        if ((!own && paged_overlap(to, {q, in * qw, in * ldq}, n_tokens)) || paged_overlap(to, {k, in * kvw, in * ldk}, n_tokens) ||
            paged_overlap(to, {v, in * kvw, in * ldv}, n_tokens))
            return paged_fail(ABRA_E_INVALID, "q_out must not share the memory of q, k or v");
    }
    if (rope && rope_len < 1) return paged_fail(ABRA_E_INVALID, "rope_len must be positive");
    const int64_t heads = (q ? n_heads : 0) + 2ll * kv->n_kv_heads;
    if (heads > 65535) return paged_fail(ABRA_E_UNSUPPORTED, "over 65535 heads of a token");
    AppendArgs p{paged_view(kv), q, k, v, ldq, ldk, ldv, ldqo, cu_new, q_norm, k_norm, rope, q_out, eps, n_heads, n_tokens, rope_len,
                 // few tokens: one a CTA, for the shortest way; many: the lookups shared
                 n_tokens >= 8 * 148 ? APPEND_TOKENS : 1, fast_div(static_cast<uint32_t>(heads))};
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
