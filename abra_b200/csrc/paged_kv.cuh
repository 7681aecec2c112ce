// paged_kv.cuh -- the paged key-value cache as the kernels see it: address
// arithmetic, the bounds checks of what the device reads (lengths, page
// numbers), 16-bit types, and the argument checks its entry points share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "../../include/abra_b200.h"
#include "common.cuh"
#include "kernels.cuh"

namespace abra {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery's
// round-up method): s = ceil(log2 d), mul = floor(2^32 (2^s - d) / d) + 1.
struct FastDiv {
    uint32_t d, mul, shift;
    __device__ __forceinline__ int div(int n) const {
        return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
    }
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

// abra_paged_kv with its page division; passed to kernels by value.
struct PagedKv {
    abra_paged_kv a;
    FastDiv page;
};

// What a step's earlier kernels may have written (lengths, tables, queries) is
// read with ordinary loads: these kernels start before the one in front of them
// has ended, and the read-only path asks for data that stays as it is from then
// on.

// Slots of sequence s, clamped to what the table can name.
__device__ __forceinline__ int paged_len(const PagedKv &kv, int s) {
    const int n = kv.a.lens[s], cap = kv.a.max_pages * kv.a.page_size;
    if (n >= 0 && n <= cap) return n;
    report_error(ERR_BAD_INDEX);
    return n < 0 ? 0 : cap;
}
__device__ __forceinline__ int paged_next_pos(const PagedKv &kv, int s, int len) {
    return kv.a.next_pos ? kv.a.next_pos[s] : len;
}
// Page number of table entry p of sequence s; -1 (and the error bit) when it
// is outside the pool.
__device__ __forceinline__ int paged_page(const PagedKv &kv, int s, int p) {
    const int page = kv.a.table[static_cast<int64_t>(s) * kv.a.table_stride + p];
    if (static_cast<unsigned>(page) < static_cast<unsigned>(kv.a.n_pages)) return page;
    report_error(ERR_BAD_INDEX);
    return -1;
}
__device__ __forceinline__ int64_t paged_k_at(const PagedKv &kv, int page, int head, int off) {
    return page * kv.a.k_page_stride + head * kv.a.k_head_stride + off * kv.a.k_slot_stride;
}
__device__ __forceinline__ int64_t paged_v_at(const PagedKv &kv, int page, int head, int off) {
    return page * kv.a.v_page_stride + head * kv.a.v_head_stride + off * kv.a.v_slot_stride;
}
// Index into acc and pos.
__device__ __forceinline__ int64_t paged_meta_at(const PagedKv &kv, int page, int head, int off) {
    return (static_cast<int64_t>(page) * kv.a.n_kv_heads + head) * kv.a.page_size + off;
}

// 16-bit types
template <typename T> struct Half16;
template <> struct Half16<__half> {
    static constexpr int type = ABRA_GGML_F16;
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Half16<__nv_bfloat16> {
    static constexpr int type = ABRA_GGML_BF16;
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

// ------------------------------------------------------------------ host ---
inline int paged_fail(int code, const char *fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return record_failure(code, msg);
}
inline bool paged_aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows in memory: `width` bytes every `stride`.
struct PagedRows {
    const void *at;
    int64_t width, stride;
};
// Whether two tensors of n rows share memory.  Columns of the same wider rows do
// not, though they lie in one range.
inline bool paged_overlap(PagedRows a, PagedRows b, int64_t n) {
    const __int128 a0 = reinterpret_cast<uintptr_t>(a.at), b0 = reinterpret_cast<uintptr_t>(b.at);
    const __int128 a1 = a0 + static_cast<__int128>(n - 1) * a.stride + a.width, b1 = b0 + static_cast<__int128>(n - 1) * b.stride + b.width;
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.stride != b.stride) return true;
    const __int128 gap = b0 >= a0 ? (b0 - a0) % a.stride : (a.stride - (a0 - b0) % a.stride) % a.stride;  // from a's columns to b's
    return gap < a.width || gap + b.width > a.stride;
}

// The checks every entry point makes of the cache it is given.
inline int paged_check(const abra_paged_kv *kv) {
    if (!kv) return paged_fail(ABRA_E_INVALID, "null cache");
    const bool some = kv->n_seqs > 0;  // no sequences need no table
    if (kv->n_seqs < 0 || kv->n_pages < 1 || kv->n_kv_heads < 1 || kv->page_size < 1 || kv->max_pages < (some ? 1 : 0))
        return paged_fail(ABRA_E_INVALID,
                          "n_seqs must not be negative, n_pages, n_kv_heads, page_size and max_pages positive "
                          "(%d, %d, %d, %d, %d)",
                          kv->n_seqs, kv->n_pages, kv->n_kv_heads, kv->page_size, kv->max_pages);
    if (static_cast<int64_t>(kv->max_pages) * kv->page_size > (1 << 30))
        return paged_fail(ABRA_E_UNSUPPORTED, "max_pages * page_size over 2^30 slots");
    if (kv->n_kv_heads > 65535 || kv->n_seqs > 65535)
        return paged_fail(ABRA_E_UNSUPPORTED, "over 65535 sequences or kv heads");
    if (kv->head_dim != 64 && kv->head_dim != 96 && kv->head_dim != 128)
        return paged_fail(ABRA_E_UNSUPPORTED, "head_dim must be 64, 96 or 128 (got %d)", kv->head_dim);
    if (kv->type != ABRA_GGML_F16 && kv->type != ABRA_GGML_BF16)
        return paged_fail(ABRA_E_UNSUPPORTED, "the cache's type must be F16 or BF16 (got %d)", kv->type);
    if (!kv->k || !kv->v || (some && (!kv->table || !kv->lens))) return paged_fail(ABRA_E_INVALID, "null pointer in the cache");
    if (!paged_aligned(kv->k, 16) || !paged_aligned(kv->v, 16))
        return paged_fail(ABRA_E_INVALID, "the pools must be 16-byte aligned");
    if (!paged_aligned(kv->acc, 4) || !paged_aligned(kv->pos, 4) || !paged_aligned(kv->table, 4) ||
        !paged_aligned(kv->lens, 4) || !paged_aligned(kv->next_pos, 4))
        return paged_fail(ABRA_E_INVALID, "acc, pos, table, lens and next_pos must be 4-byte aligned");
    const int64_t strides[] = {kv->k_page_stride, kv->k_head_stride, kv->k_slot_stride,
                               kv->v_page_stride, kv->v_head_stride, kv->v_slot_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return paged_fail(ABRA_E_INVALID, "strides must be multiples of 8 elements (got %lld)", (long long)s);
    if (kv->table_stride < kv->max_pages) return paged_fail(ABRA_E_INVALID, "table_stride < max_pages");
    return ABRA_OK;
}
inline PagedKv paged_view(const abra_paged_kv *kv) { return {*kv, fast_div(static_cast<uint32_t>(kv->page_size))}; }
// Sets a kernel's dynamic shared memory limit once a device (bit d of `done`).
inline cudaError_t paged_smem(const void *k, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (done.load(std::memory_order_relaxed) >> (dev & 63) & 1)) return e;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return e;
}
// A launch that may begin before the kernel in front of it in the stream has
// ended; the kernel's pdl_wait, ahead of everything it reads, waits for that.
// Clusters of `cluster` CTAs along x, or none (0).
inline cudaError_t paged_launch(const void *k, dim3 grid, int threads, int smem, cudaStream_t st, void **args, int cluster = 0) {
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, k, args);
}
template <typename Args> cudaError_t paged_launch(void (*k)(Args), dim3 grid, int threads, int smem, cudaStream_t st, Args a) {
    void *args[] = {&a};
    return paged_launch(reinterpret_cast<const void *>(k), grid, threads, smem, st, args);
}
inline int paged_cuda(cudaError_t e, const char *what) {
    return e == cudaSuccess ? ABRA_OK : paged_fail(ABRA_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace abra
