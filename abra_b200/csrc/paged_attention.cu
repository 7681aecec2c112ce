// paged_attention.cu -- attention of each sequence's newest tokens over its
// paged key-value cache, with the slots' accumulated weights
// (abra_paged_attention).
//
// For query j of n_q, q head h of kv head g: s_t = scale q.k_t over the slots t
// < len - (n_q - 1 - j), lse = log sum_t exp s_t, out = sum_t exp(s_t - lse)
// v_t; acc_t += exp(s_t - lse) over the group's heads and the n_q queries.
#include "paged_kv.cuh"

namespace abra {
namespace {

struct AttendArgs {
    PagedKv kv;
    const void *q;
    void *out;
    float *lse, *rows_lse;  // lse of every row for the accumulation (workspace)
    int64_t ldq, ldo;
    float scale;
    int n_heads, n_q, accumulate, out_f32;
};

constexpr int AT_WARPS = 8;

// One CTA per (kv head, sequence); its rows (query, head of the group) in
// turn, the warps taking every eighth slot with a running maximum and sum of
// their own; lane l holds the elements l, l + 32, ...
template <typename T, int D>
__global__ void __launch_bounds__(AT_WARPS * 32) attend_kernel(const __grid_constant__ AttendArgs p) {
    constexpr int N = D / 32;
    __shared__ float s_m[AT_WARPS], s_l[AT_WARPS], s_o[AT_WARPS][D];
    const int g = blockIdx.x, s = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = p.n_heads / p.kv.a.n_kv_heads, rows = group * p.n_q;
    const int len = paged_len(p.kv, s);
    const T *kp = static_cast<const T *>(p.kv.a.k), *vp = static_cast<const T *>(p.kv.a.v);
    float *row_lse = p.rows_lse + (static_cast<int64_t>(s) * gridDim.x + g) * rows;

    for (int r = 0; r < rows; ++r) {
        const int j = r / group, h = g * group + r % group;
        const int seen = len - (p.n_q - 1 - j);
        const int64_t row = static_cast<int64_t>(s) * p.n_q + j;
        const T *q = static_cast<const T *>(p.q) + row * p.ldq + static_cast<int64_t>(h) * D;
        float qf[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) qf[i] = Half16<T>::up(q[lane + 32 * i]) * p.scale, o[i] = 0.0f;
        for (int t = warp; t < seen; t += AT_WARPS) {
            const int e = p.kv.page.div(t), off = t - e * p.kv.a.page_size;
            const int page = max(0, paged_page(p.kv, s, e));
            const T *k = kp + paged_k_at(p.kv, page, g, off), *v = vp + paged_v_at(p.kv, page, g, off);
            float sc = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) sc += qf[i] * Half16<T>::up(k[lane + 32 * i]);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, x);
            const float mn = fmaxf(m, sc), a = expf(m - mn), w = expf(sc - mn);
            l = l * a + w;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = o[i] * a + w * Half16<T>::up(v[lane + 32 * i]);
            m = mn;
        }
        if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
        for (int i = 0; i < N; ++i) s_o[warp][lane + 32 * i] = o[i];
        __syncthreads();
        float top = s_m[0], total = 0.0f;
        for (int w = 1; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w]);
        for (int w = 0; w < AT_WARPS; ++w) total += s_l[w] != 0.0f ? s_l[w] * expf(s_m[w] - top) : 0.0f;
        const float lse = seen > 0 ? top + logf(total) : -INFINITY;
        if (threadIdx.x == 0) {
            row_lse[r] = lse;
            if (p.lse) p.lse[row * p.n_heads + h] = lse;
        }
        for (int d = threadIdx.x; d < D; d += AT_WARPS * 32) {
            float sum = 0.0f;
            for (int w = 0; w < AT_WARPS; ++w) sum += s_l[w] != 0.0f ? s_o[w][d] * expf(s_m[w] - top) : 0.0f;
            const float x = seen > 0 ? sum / total : 0.0f;
            const int64_t at = row * p.ldo + static_cast<int64_t>(h) * D + d;
            if (p.out_f32) static_cast<float *>(p.out)[at] = x;
            else static_cast<T *>(p.out)[at] = Half16<T>::down(x);
        }
        __syncthreads();
    }
    if (!p.accumulate) return;
    for (int t = warp; t < len; t += AT_WARPS) {
        const int e = p.kv.page.div(t), off = t - e * p.kv.a.page_size;
        const int page = paged_page(p.kv, s, e);
        if (page < 0) continue;
        const T *k = kp + paged_k_at(p.kv, page, g, off);
        float sum = 0.0f;
        for (int r = 0; r < rows; ++r) {
            const int j = r / group, h = g * group + r % group;
            const T *q = static_cast<const T *>(p.q) + (static_cast<int64_t>(s) * p.n_q + j) * p.ldq + static_cast<int64_t>(h) * D;
            float sc = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) sc += Half16<T>::up(q[lane + 32 * i]) * p.scale * Half16<T>::up(k[lane + 32 * i]);
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, x);
            if (t < len - (p.n_q - 1 - j)) sum += expf(sc - row_lse[r]);
        }
        if (lane == 0) p.kv.a.acc[paged_meta_at(p.kv, page, g, off)] += sum;
    }
}

template <typename T>
cudaError_t launch(const AttendArgs &p, cudaStream_t st) {
    const dim3 grid(p.kv.a.n_kv_heads, p.kv.a.n_seqs);
    switch (p.kv.a.head_dim) {
        case 64: attend_kernel<T, 64><<<grid, AT_WARPS * 32, 0, st>>>(p); break;
        case 96: attend_kernel<T, 96><<<grid, AT_WARPS * 32, 0, st>>>(p); break;
        default: attend_kernel<T, 128><<<grid, AT_WARPS * 32, 0, st>>>(p); break;
    }
    return cudaGetLastError();
}

int check(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q, int32_t flags) {
    const int rc = paged_check(kv);
    if (rc) return rc;
    if (n_heads < 1 || n_heads > 65535 || n_heads % kv->n_kv_heads)
        return paged_fail(ABRA_E_INVALID, "n_heads (%d) must be a multiple of the %d kv heads", n_heads, kv->n_kv_heads);
    if (n_q < 1 || n_q > 4096) return paged_fail(ABRA_E_INVALID, "n_q must be 1 to 4096 (got %d)", n_q);
    if (flags & ~ABRA_PAGED_ACCUMULATE) return paged_fail(ABRA_E_INVALID, "unknown flags %d", flags);
    if ((flags & ABRA_PAGED_ACCUMULATE) && !kv->acc) return paged_fail(ABRA_E_INVALID, "accumulation needs acc");
    return ABRA_OK;
}

int64_t workspace_bytes_of(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q) {
    return 256 + static_cast<int64_t>(kv->n_seqs) * n_heads * n_q * 4;
}

}  // namespace
}  // namespace abra

ABRA_ERROR_WORD_ACCESSOR(paged_attention_error_word)

extern "C" int64_t abra_paged_attention_workspace(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q,
                                                  int32_t flags) {
    const int rc = abra::check(kv, n_heads, n_q, flags);
    return rc ? rc : abra::workspace_bytes_of(kv, n_heads, n_q);
}

extern "C" int abra_paged_attention(const abra_paged_kv *kv, const void *q, int64_t ldq, int32_t n_heads,
                                    int32_t n_q, float scale, void *out, int32_t out_type, int64_t ldo,
                                    float *lse, int32_t flags, void *workspace, int64_t workspace_bytes,
                                    void *stream) {
    using namespace abra;
    const int rc = check(kv, n_heads, n_q, flags);
    if (rc) return rc;
    if (out_type != kv->type && out_type != ABRA_GGML_F32)
        return paged_fail(ABRA_E_UNSUPPORTED, "out must be of the cache's type or F32 (got %d)", out_type);
    if (!q || !out || !workspace) return paged_fail(ABRA_E_INVALID, "null q, out or workspace");
    if (ldq < static_cast<int64_t>(n_heads) * kv->head_dim || ldo < static_cast<int64_t>(n_heads) * kv->head_dim)
        return paged_fail(ABRA_E_INVALID, "a row stride is smaller than its heads");
    if (ldq % 8 || ldo % 8 || !paged_aligned(q, 16) || !paged_aligned(out, 16) || !paged_aligned(lse, 4))
        return paged_fail(ABRA_E_INVALID, "q and out rows must start on 16 bytes and their strides be multiples of 8 elements");
    if (!paged_aligned(workspace, 256)) return paged_fail(ABRA_E_INVALID, "the workspace must be 256-byte aligned");
    if (workspace_bytes < workspace_bytes_of(kv, n_heads, n_q))
        return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                          (long long)workspace_bytes_of(kv, n_heads, n_q));
    if (kv->n_seqs == 0) return ABRA_OK;
    AttendArgs p{paged_view(kv), q, out, lse, reinterpret_cast<float *>(static_cast<char *>(workspace) + 256), ldq, ldo,
                 scale, n_heads, n_q, flags & ABRA_PAGED_ACCUMULATE, out_type == ABRA_GGML_F32};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return paged_cuda(kv->type == ABRA_GGML_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st),
                      "paged attention launch");
}
