// paged_evict.cu -- eviction from a paged key-value cache by accumulated
// weight (abra_paged_evict).
//
// Every (sequence, kv head) with more than `budget` slots ranks them by a
// 32-bit key -- protected slots (first positions, recent positions) above all,
// the others in the order of their weight -- and keeps the `budget` largest,
// ties to the lowest slot.  Only rows that have to move do: the i-th evicted
// slot below the budget takes the i-th kept one above it, so sources (slots >=
// budget) and targets (< budget) never meet and the order of the copies does
// not matter.
#include "paged_kv.cuh"

namespace abra {
namespace {

struct EvictArgs {
    PagedKv kv;
    int32_t *new_lens, *moves;
    int budget, n_sink, n_recent, cap;  // cap: entries of a move list
};

// Unsigned order of the weights: the float's bits with the sign folded, -0 as
// 0, NaN as -infinity; protected slots get the largest key of all.
__device__ __forceinline__ uint32_t rank_key(float a, int pos, int n_sink, int recent_from) {
    if (pos < n_sink || pos >= recent_from) return 0xffffffffu;
    if (a != a) a = -INFINITY;
    const uint32_t u = __float_as_uint(a + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int EV_THREADS = 256;

__device__ __forceinline__ int block_sum(int v, int *buf) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) t += buf[w];
    return t;
}
// Exclusive rank of this thread's flag in the block; *total gets the count.
__device__ __forceinline__ int block_rank(bool f, int *buf, int *total) {
    const unsigned b = __ballot_sync(0xffffffffu, f);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) buf[warp] = __popc(b);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) {
        if (w < warp) before += buf[w];
        all += buf[w];
    }
    *total = all;
    return before + __popc(b & ((1u << lane) - 1u));
}

// One CTA per (kv head, sequence): the budget-th largest key bit by bit, then
// one walk over the slots that lists holes and movers, then the copies.
template <int D>
__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const __grid_constant__ EvictArgs p) {
    __shared__ int buf[EV_THREADS / 32];
    const int g = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int len = paged_len(p.kv, s);
    if (g == 0 && tid == 0) p.new_lens[s] = min(len, p.budget);
    if (len <= p.budget) return;
    const int recent_from = paged_next_pos(p.kv, s, len) - p.n_recent;
    auto meta = [&](int t) {
        const int e = p.kv.page.div(t);
        return paged_meta_at(p.kv, max(0, paged_page(p.kv, s, e)), g, t - e * p.kv.a.page_size);
    };
    auto key = [&](int t) {
        const int64_t m = meta(t);
        return rank_key(p.kv.a.acc[m], p.kv.a.pos[m], p.n_sink, recent_from);
    };
    uint32_t cut = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = cut | (1u << bit);
        int n = 0;
        for (int t = tid; t < len; t += EV_THREADS) n += key(t) >= c;
        if (block_sum(n, buf) >= p.budget) cut = c;
    }
    int above = 0;
    for (int t = tid; t < len; t += EV_THREADS) above += key(t) > cut;
    const int ties = p.budget - block_sum(above, buf);  // this many slots with the key `cut` stay
    int32_t *hole = p.moves + (static_cast<int64_t>(s) * p.kv.a.n_kv_heads + g) * 2 * p.cap, *mover = hole + p.cap;
    int n_tie = 0, n_hole = 0, n_mover = 0;
    for (int t0 = 0; t0 < len; t0 += EV_THREADS) {
        const int t = t0 + tid;
        const uint32_t k = t < len ? key(t) : 0u;
        int total;
        const bool tie = t < len && k == cut;
        const int r = n_tie + block_rank(tie, buf, &total);
        n_tie += total;
        const bool keep = t < len && (k > cut || (tie && r < ties));
        const bool is_hole = t < p.budget && !keep, is_mover = t >= p.budget && keep;
        const int rh = n_hole + block_rank(is_hole, buf, &total);
        n_hole += total;
        const int rm = n_mover + block_rank(is_mover, buf, &total);
        n_mover += total;
        if (is_hole) hole[rh] = t;
        if (is_mover) mover[rm] = t;
    }
    __syncthreads();
    for (int i = tid >> 5; i < n_hole; i += EV_THREADS / 32) {
        const int lane = tid & 31, from = mover[i], to = hole[i];
        const int ef = p.kv.page.div(from), et = p.kv.page.div(to);
        const int pf = paged_page(p.kv, s, ef), pt = paged_page(p.kv, s, et);
        if (pf < 0 || pt < 0) continue;
        const int of = from - ef * p.kv.a.page_size, ot = to - et * p.kv.a.page_size;
        uint16_t *kp = static_cast<uint16_t *>(p.kv.a.k), *vp = static_cast<uint16_t *>(p.kv.a.v);
        for (int d = lane; d < D; d += 32) {
            kp[paged_k_at(p.kv, pt, g, ot) + d] = kp[paged_k_at(p.kv, pf, g, of) + d];
            vp[paged_v_at(p.kv, pt, g, ot) + d] = vp[paged_v_at(p.kv, pf, g, of) + d];
        }
        if (lane == 0) {
            const int64_t a = paged_meta_at(p.kv, pt, g, ot), b = paged_meta_at(p.kv, pf, g, of);
            p.kv.a.acc[a] = p.kv.a.acc[b];
            p.kv.a.pos[a] = p.kv.a.pos[b];
        }
    }
}

int check(const abra_paged_kv *kv, int32_t budget) {
    const int rc = paged_check(kv);
    if (rc) return rc;
    if (budget < 1) return paged_fail(ABRA_E_INVALID, "budget must be positive (got %d)", budget);
    return ABRA_OK;
}
// A sequence of L slots moves at most min(budget, L - budget) rows.
int64_t move_cap(const abra_paged_kv *kv, int32_t budget) {
    const int64_t slots = static_cast<int64_t>(kv->max_pages) * kv->page_size;
    return slots <= budget ? 0 : slots - budget < budget ? slots - budget : budget;
}
int64_t workspace_bytes_of(const abra_paged_kv *kv, int32_t budget) {
    return 16 + static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads * 2 * move_cap(kv, budget) * 4;
}

}  // namespace
}  // namespace abra

ABRA_ERROR_WORD_ACCESSOR(paged_evict_error_word)

extern "C" int64_t abra_paged_evict_workspace(const abra_paged_kv *kv, int32_t budget) {
    const int rc = abra::check(kv, budget);
    return rc ? rc : abra::workspace_bytes_of(kv, budget);
}

extern "C" int abra_paged_evict(const abra_paged_kv *kv, int32_t budget, int32_t n_sink, int32_t n_recent,
                                int32_t *new_lens, void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace abra;
    const int rc = check(kv, budget);
    if (rc) return rc;
    if (n_sink < 0 || n_recent < 0 || static_cast<int64_t>(n_sink) + n_recent > budget)
        return paged_fail(ABRA_E_INVALID, "n_sink (%d) and n_recent (%d) must not be negative and fit the budget (%d)", n_sink,
                          n_recent, budget);
    if (!kv->acc || !kv->pos) return paged_fail(ABRA_E_INVALID, "eviction needs acc and pos");
    if (!new_lens || !workspace) return paged_fail(ABRA_E_INVALID, "null new_lens or workspace");
    if (new_lens < kv->lens + kv->n_seqs && kv->lens < new_lens + kv->n_seqs)
        return paged_fail(ABRA_E_INVALID, "new_lens must not overlap lens");
    if (!paged_aligned(workspace, 16) || !paged_aligned(new_lens, 4))
        return paged_fail(ABRA_E_INVALID, "the workspace must be 16-byte, new_lens 4-byte aligned");
    if (workspace_bytes < workspace_bytes_of(kv, budget))
        return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                          (long long)workspace_bytes_of(kv, budget));
    if (kv->n_seqs == 0) return ABRA_OK;
    EvictArgs p{paged_view(kv), new_lens, static_cast<int32_t *>(workspace), budget, n_sink, n_recent,
                static_cast<int>(move_cap(kv, budget))};
    const dim3 grid(kv->n_kv_heads, kv->n_seqs);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (kv->head_dim) {
        case 64: evict_kernel<64><<<grid, EV_THREADS, 0, st>>>(p); break;
        case 96: evict_kernel<96><<<grid, EV_THREADS, 0, st>>>(p); break;
        default: evict_kernel<128><<<grid, EV_THREADS, 0, st>>>(p); break;
    }
    return paged_cuda(cudaGetLastError(), "paged evict launch");
}
