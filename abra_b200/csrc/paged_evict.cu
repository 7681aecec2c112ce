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
//
// Two kernels.  The first selects: a cluster of CTAs per (sequence, kv head)
// reads weights and positions once, keeps the keys in shared memory, finds the
// budget-th largest by four passes of 8 bits over them (histograms added up
// through the cluster's shared memory) and writes the lists of holes and movers
// in slot order.  The second copies, a CTA for every 128 moves of a list.
//
// Bound: 8 bytes a slot to choose among and the moved rows, read and written.
// Measured (B200, 1965 MHz, 8 kv heads of 128): one sequence of 131,072 slots to
// 32,768, 213 MB, 66 us, 27 of them the selection on 64 multiprocessors and 38
// the copies (5.3 TB/s); 32 prompts of up to 8,192 to 2,048, 126 MB, 43 us, 16
// and 20; one page over 4,096 slots 16 us, all of it the chain of the selection
// (3 us to the keys, 1.5 a radix pass, 4 for the lists) and a launch.
#include <algorithm>

#include "paged_kv.cuh"

namespace abra {
namespace {

struct EvictArgs {
    PagedKv kv;
    int32_t *new_lens, *counts, *moves;  // counts: moves of a row; moves: its holes, then its movers, cap each
    int budget, n_sink, n_recent, cap, held;  // held: keys of a CTA that fit its shared memory
};

// Unsigned order of the weights: the float's bits with the sign folded, -0 as
// 0, NaN as -infinity; protected slots get the largest key of all.
__device__ __forceinline__ uint32_t rank_key(float a, int pos, int n_sink, int recent_from) {
    if (pos < n_sink || pos >= recent_from) return 0xffffffffu;
    if (a != a) a = -INFINITY;
    const uint32_t u = __float_as_uint(a + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int cluster_rank() {
    int r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int cluster_size() {
    int n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
constexpr int MOST_CTAS = 8;  // of a cluster
// What CTA `rank` of the cluster has at this address of its shared memory.
__device__ __forceinline__ int peer_value(const int *p, int rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ int4 peer_value4(const int4 *p, int rank) {
    uint32_t at;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32;
static_assert(SEL_WARPS == 32, "lanes stand for warps");
constexpr int BINS = 256;
constexpr int LANE_BINS_BYTES = BINS * 32 * 4;

// One cluster per (kv head, sequence), an equal run of slots for each CTA.
__global__ void __launch_bounds__(SEL_THREADS) select_kernel(const __grid_constant__ EvictArgs p) {
    extern __shared__ __align__(16) unsigned char smem[];
    int *bins = reinterpret_cast<int *>(smem);  // [BINS][32 lanes]: a lane's own column, so equal keys do not collide
    uint32_t *held = reinterpret_cast<uint32_t *>(smem + LANE_BINS_BYTES);  // keys of the first p.held slots
    __shared__ __align__(16) int s_hist[2][BINS];
    __shared__ int s_found[3], s_tie[SEL_WARPS], s_hole[SEL_WARPS], s_mover[SEL_WARPS], s_total[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster_rank(), size = cluster_size();
    const int g = blockIdx.y, s = blockIdx.z;
    pdl_wait();
    pdl_launch_dependents();
    const int len = paged_len(p.kv, s);
    const int64_t row = static_cast<int64_t>(s) * p.kv.a.n_kv_heads + g;
    if (rank == 0 && tid == 0) {
        if (g == 0) p.new_lens[s] = min(len, p.budget);
        if (len <= p.budget) p.counts[row] = 0;
    }
    if (len <= p.budget) return;  // the whole cluster
    const int recent_from = paged_next_pos(p.kv, s, len) - p.n_recent;
    const int per = (len + size - 1) / size, first = min(len, rank * per), n = min(len, first + per) - first;
    auto load_key = [&](int t) {
        const int e = p.kv.page.div(t);
        const int64_t m = paged_meta_at(p.kv, max(0, paged_page(p.kv, s, e)), g, t - e * p.kv.a.page_size);
        return rank_key(__ldcg(p.kv.a.acc + m), __ldcg(p.kv.a.pos + m), p.n_sink, recent_from);
    };
    auto key = [&](int i) { return i < p.held ? held[i] : load_key(first + i); };
    for (int i = tid; i < BINS * 32; i += SEL_THREADS) bins[i] = 0;
#pragma unroll 8
    for (int i = tid; i < min(n, p.held); i += SEL_THREADS) held[i] = load_key(first + i);
    __syncthreads();

    // ---- the budget-th largest key, 8 bits at a time, until all keys with the
    // leading bits found so far are kept or they are the whole key ----
    uint32_t cut = 0;
    int left = p.budget, same = 0, pass = 0;  // of the `same` keys that share cut's leading bits, `left` are kept
#pragma unroll 1
    for (; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
#pragma unroll 4
        for (int i = tid; i < n; i += SEL_THREADS) {
            const uint32_t k = key(i);
            if (pass == 0 || (k >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&bins[((k >> shift) & 255) * 32 + lane], 1);
        }
        __syncthreads();
        int *hist = s_hist[pass & 1];
        if (tid < BINS) {
            int sum = 0;
#pragma unroll
            for (int x = 0; x < 32; ++x) sum += bins[tid * 32 + ((x + tid) & 31)];
            hist[tid] = sum;
        }
        if (size > 1) cluster_sync();
        else __syncthreads();
        if (warp == 0) {  // lane l: bins 8 l .. 8 l + 7 of all CTAs; a scan from the top bin
            int b[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < MOST_CTAS; ++r)
                if (r < size) {
                    const int4 x = peer_value4(reinterpret_cast<const int4 *>(hist) + 2 * lane, r);
                    const int4 y = peer_value4(reinterpret_cast<const int4 *>(hist) + 2 * lane + 1, r);
                    b[0] += x.x, b[1] += x.y, b[2] += x.z, b[3] += x.w, b[4] += y.x, b[5] += y.y, b[6] += y.z, b[7] += y.w;
                }
            int above = b[0] + b[1] + b[2] + b[3] + b[4] + b[5] + b[6] + b[7];
            const int own = above;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_down_sync(0xffffffffu, above, d);
                if (lane + d < 32) above += y;
            }
            above -= own;  // keys in higher lanes' bins
#pragma unroll
            for (int x = 7; x >= 0; --x) {
                if (above < left && above + b[x] >= left) s_found[0] = 8 * lane + x, s_found[1] = left - above, s_found[2] = b[x];
                above += b[x];
            }
        } else {  // the others empty the bins for the next pass
            for (int i = tid - 32; i < BINS * 32; i += SEL_THREADS - 32) bins[i] = 0;
        }
        __syncthreads();
        cut |= static_cast<uint32_t>(s_found[0]) << shift;
        left = s_found[1], same = s_found[2];
        if (left == same) break;  // the same in every CTA
    }
    // Slots with a key above cut stay, and of those at cut the lowest `left`.
    // Only after four passes can there be others at cut (equal keys); the last
    // pass counted them in each CTA.
    const bool equals = left != same;
    int ties = 0;

    // ---- holes and movers in slot order: a run of slots for each warp ----
    const int run = ((n + SEL_WARPS - 1) / SEL_WARPS + 31) & ~31, w0 = min(n, warp * run), w1 = min(n, w0 + run);
    if (equals) {
        for (int r = 0; r < rank; ++r) ties += peer_value(&s_hist[1][cut & 255], r);
        int own = 0;
#pragma unroll 4
        for (int i = w0; i < w1; i += 32) own += __popc(__ballot_sync(0xffffffffu, i + lane < w1 && key(i + lane) == cut));
        if (lane == 0) s_tie[warp] = own;
        __syncthreads();
        for (int x = 0; x < warp; ++x) ties += s_tie[x];
    }
    // one step of 32 slots: which are holes, which movers
    const unsigned below = (1u << lane) - 1u;
    auto classify = [&](int i, int &tie, unsigned &holes, unsigned &movers) {
        const bool in = i + lane < w1;
        const uint32_t k = in ? key(i + lane) : 0u;
        bool keep = in && k >= cut;
        if (equals) {
            const unsigned t = __ballot_sync(0xffffffffu, in && k == cut);
            keep = in && (k > cut || (k == cut && tie + __popc(t & below) < left));
            tie += __popc(t);
        }
        const bool low = first + i + lane < p.budget;
        holes = __ballot_sync(0xffffffffu, in && low && !keep);
        movers = __ballot_sync(0xffffffffu, !low && keep);
    };
    int nh = 0, nm = 0, tie = ties;
#pragma unroll 4
    for (int i = w0; i < w1; i += 32) {
        unsigned h, m;
        classify(i, tie, h, m);
        nh += __popc(h), nm += __popc(m);
    }
    if (lane == 0) s_hole[warp] = nh, s_mover[warp] = nm;
    __syncthreads();
    // lanes add up the warps, and the CTAs of the cluster
    int hole_at = s_hole[lane], mover_at = s_mover[lane];
    if (warp == 0) {
        const int h = __reduce_add_sync(0xffffffffu, hole_at), m = __reduce_add_sync(0xffffffffu, mover_at);
        if (lane == 0) s_total[0] = h, s_total[1] = m;
    }
    hole_at = __reduce_add_sync(0xffffffffu, lane < warp ? hole_at : 0);
    mover_at = __reduce_add_sync(0xffffffffu, lane < warp ? mover_at : 0);
    if (size > 1) cluster_sync();
    else __syncthreads();
    hole_at += __reduce_add_sync(0xffffffffu, lane < rank ? peer_value(&s_total[0], lane) : 0);
    mover_at += __reduce_add_sync(0xffffffffu, lane < rank ? peer_value(&s_total[1], lane) : 0);
    if (rank == size - 1 && tid == 0) p.counts[row] = hole_at + s_total[0];
    int32_t *hole = p.moves + row * 2 * p.cap, *mover = hole + p.cap;
    tie = ties;
#pragma unroll 4
    for (int i = w0; i < w1; i += 32) {
        unsigned h, m;
        classify(i, tie, h, m);
        if (h >> lane & 1) hole[hole_at + __popc(h & below)] = first + i + lane;
        if (m >> lane & 1) mover[mover_at + __popc(m & below)] = first + i + lane;
        hole_at += __popc(h), mover_at += __popc(m);
    }
    if (size > 1) cluster_sync();  // nobody leaves while its shared memory is read
}

constexpr int MOVE_THREADS = 256, MOVES = 128;

// MOVES moves of one list: the addresses first, then 16-byte copies, several in
// flight a thread.  A CTA for each 128 moves that a list may have at most, most
// of them empty, ends sooner than four CTAs a multiprocessor that share all
// moves equally (47 against 54 us for 118 MB of 128 lists): equal bytes do not
// take equal times.
template <int D>
__global__ void __launch_bounds__(MOVE_THREADS, 4) move_kernel(const __grid_constant__ EvictArgs p) {
    constexpr int CH = D / 8;  // 16-byte chunks of a row
    constexpr int BATCH = 8;
    __shared__ int64_t s_from[2][MOVES], s_to[2][MOVES];  // K, V
    __shared__ bool s_ok[MOVES];
    const int g = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const int64_t row = static_cast<int64_t>(s) * p.kv.a.n_kv_heads + g;
    pdl_wait();
    pdl_launch_dependents();
    const int first = blockIdx.x * MOVES, n = min(MOVES, __ldcg(p.counts + row) - first);
    if (n <= 0) return;
    const int32_t *hole = p.moves + row * 2 * p.cap + first, *mover = hole + p.cap;
    if (tid < n) {
        const int from = __ldcg(mover + tid), to = __ldcg(hole + tid);
        const int ef = p.kv.page.div(from), et = p.kv.page.div(to);
        const int pf = paged_page(p.kv, s, ef), pt = paged_page(p.kv, s, et);
        const int of = from - ef * p.kv.a.page_size, ot = to - et * p.kv.a.page_size;
        s_ok[tid] = pf >= 0 && pt >= 0;
        if (s_ok[tid]) {
            s_from[0][tid] = paged_k_at(p.kv, pf, g, of), s_to[0][tid] = paged_k_at(p.kv, pt, g, ot);
            s_from[1][tid] = paged_v_at(p.kv, pf, g, of), s_to[1][tid] = paged_v_at(p.kv, pt, g, ot);
            const int64_t a = paged_meta_at(p.kv, pt, g, ot), b = paged_meta_at(p.kv, pf, g, of);
            p.kv.a.acc[a] = p.kv.a.acc[b];
            p.kv.a.pos[a] = p.kv.a.pos[b];
        }
    }
    __syncthreads();
    for (int x0 = tid; x0 < n * 2 * CH; x0 += BATCH * MOVE_THREADS) {
        uint4 v[BATCH];
        uint16_t *to[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int x = x0 + b * MOVE_THREADS, m = x / (2 * CH), kv = (x / CH) & 1, chunk = x % CH;
            to[b] = nullptr;
            if (x < n * 2 * CH && s_ok[m]) {
                uint16_t *pool = static_cast<uint16_t *>(kv ? p.kv.a.v : p.kv.a.k) + 8 * chunk;
                v[b] = __ldcg(reinterpret_cast<const uint4 *>(pool + s_from[kv][m]));
                to[b] = pool + s_to[kv][m];
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
            if (to[b]) __stcg(reinterpret_cast<uint4 *>(to[b]), v[b]);
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
int64_t rows_of(const abra_paged_kv *kv) { return static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads; }
int64_t counts_bytes(const abra_paged_kv *kv) { return (rows_of(kv) * 4 + 15) / 16 * 16 + 16; }
int64_t workspace_bytes_of(const abra_paged_kv *kv, int32_t budget) {
    return counts_bytes(kv) + rows_of(kv) * 2 * move_cap(kv, budget) * 4;
}

constexpr int HELD_MOST = 40960;  // keys in a CTA's shared memory

// CTAs of a cluster: doubled while all clusters stay resident together and
// every CTA keeps four slots a thread; adding up histograms of a cluster costs
// more than a few slots do.
int cluster_of(const abra_paged_kv *kv, int sms) {
    const int64_t slots = static_cast<int64_t>(kv->max_pages) * kv->page_size;
    int c = 1;
    while (c < MOST_CTAS && ((rows_of(kv) * c * 2 <= 2 * sms && slots / c > 4 * SEL_THREADS) || slots / c > HELD_MOST)) c *= 2;
    return c;
}

cudaError_t launch(EvictArgs &p, cudaStream_t st) {
    const int64_t slots = static_cast<int64_t>(p.kv.a.max_pages) * p.kv.a.page_size;
    const int cluster = cluster_of(&p.kv.a, device_sm_count());
    p.held = static_cast<int>(std::min<int64_t>((slots + cluster - 1) / cluster, HELD_MOST));
    const int smem = LANE_BINS_BYTES + p.held * 4;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = paged_smem(reinterpret_cast<const void *>(select_kernel), LANE_BINS_BYTES + HELD_MOST * 4, done);
    if (e != cudaSuccess) return e;
    const unsigned heads = p.kv.a.n_kv_heads, seqs = p.kv.a.n_seqs;
    void *args[] = {&p};
    e = paged_launch(reinterpret_cast<const void *>(select_kernel), dim3(cluster, heads, seqs), SEL_THREADS, smem, st, args, cluster);
    if (e != cudaSuccess || p.cap == 0) return e;
    const void *k = p.kv.a.head_dim == 64   ? reinterpret_cast<const void *>(move_kernel<64>)
                    : p.kv.a.head_dim == 96 ? reinterpret_cast<const void *>(move_kernel<96>)
                                            : reinterpret_cast<const void *>(move_kernel<128>);
    return paged_launch(k, dim3((p.cap + MOVES - 1) / MOVES, heads, seqs), MOVE_THREADS, 0, st, args);
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
    if (kv->n_seqs == 0) return ABRA_OK;
    if (!new_lens || !workspace) return paged_fail(ABRA_E_INVALID, "null new_lens or workspace");
    if (new_lens < kv->lens + kv->n_seqs && kv->lens < new_lens + kv->n_seqs)
        return paged_fail(ABRA_E_INVALID, "new_lens must not overlap lens");
    if (!paged_aligned(workspace, 16) || !paged_aligned(new_lens, 4))
        return paged_fail(ABRA_E_INVALID, "the workspace must be 16-byte, new_lens 4-byte aligned");
    if (workspace_bytes < workspace_bytes_of(kv, budget))
        return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                          (long long)workspace_bytes_of(kv, budget));
    char *ws = static_cast<char *>(workspace);
    EvictArgs p{paged_view(kv), new_lens, reinterpret_cast<int32_t *>(ws), reinterpret_cast<int32_t *>(ws + counts_bytes(kv)),
                budget, n_sink, n_recent, static_cast<int>(move_cap(kv, budget)), 0};
    return paged_cuda(launch(p, static_cast<cudaStream_t>(stream)), "paged evict launch");
}
