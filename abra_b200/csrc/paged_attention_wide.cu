// paged_attention_wide.cu -- the paged attention's kernel for many rows a kv
// head (several new tokens of a group: verification of drafts, or wide groups),
// on the 5th-generation tensor cores.
//
// With R = group x n_q rows a slot of a kv head costs 6 R D flops (the weights
// go in twice, below) for 4 D bytes: at 64 rows 96 flops a byte, 630 TFLOP/s at
// the HBM's rate.  mma.sync's pipe does 580 at most here (two cycles a 16x8x16
// product and multiprocessor), before anything else is issued; tcgen05's limit
// is the shared memory that its operands are read from, about 60 cycles for a
// 128-row one of 16 columns whatever N is, 1,440 a step of 128 slots against the
// 2,900 that the step's bytes take.
//
// A CTA takes steps of 128 slots.  Three loader warps copy K and V rows into
// rings of tiles, one warp issues the tensor core's work, and a thread of the
// four or eight compute warps stands for a slot.  Per step
//   S^T[128 slots x N] = K Q^T      (M 128, N rows, K = D)
//   P^T = 2^(S^T - m + SHIFT), split into two 16-bit values, to shared memory
//   O^T[D x N] += V^T P^T           (M 128, K = 128 slots, twice)
// with S^T (two buffers) and O^T in tensor memory, all operands in shared memory
// in rows of 128 bytes (64 elements; wider rows in planes) with the 128-byte
// swizzle: 16-byte chunk c of row r at r * 128 + (c ^ r % 8) * 16.  The same
// bytes are a K-major operand (K and Q: the chunks walk along D) and an M-major
// one (V and P: the rows are the contracted slots).  The next step's scores are
// issued as soon as its keys have landed, this step's sum as soon as its weights
// are written, by a warp in uniform control flow: issued by one thread of a
// branch, each product cost 40 to 80 ns of register moves, five times its work.
// For heads of less than 128 the O^T product also takes what lies behind V in
// shared memory: into rows beyond D of O^T that nobody reads.
//
// Measured (B200, 1965 MHz): 16 queries of 4 heads over 4 sequences of up to
// 8,192 slots 26 us (mma.sync with 32 rows a block: 68); 16 heads of one token
// over 131,072 slots, 0.54 GB, 100 us = 5.4 TB/s.  A step of 64 rows takes 1.2
// us of softmax and 1.7 of copies; a CTA's start, 3.5 us to its first scores,
// and a row's end, 2 us, run beside nothing and bound the smaller calls.  A prompt's
// blocks of rows each take all of their sequence's slots, also those that none of
// them sees: 4,096 tokens of 32 heads 1.5 ms, half of it for nothing.
#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace abra {
namespace {

constexpr int W_LOAD = 96;  // three loader warps

template <int D, int N> struct Wide {
    // compute warps: four, or eight that share the rows of a slot where these
    // are so many that four take longer than the copies (2.0 us a step of 64
    // rows; 16 queries of 4 sequences 32.0 us with four, 26.3 with eight)
    static constexpr int CW = N >= 64 ? 8 : 4, COMPUTE = 32 * CW, THREADS = COMPUTE + W_LOAD + 32;
    static constexpr int NH = N / (CW / 4);             // rows of a compute thread
    static constexpr int CHUNKS = D / 8;                // of 16 bytes in a row
    static constexpr int PLANES = (D + 63) / 64;
    static constexpr int PLANE = WIDE_STEP * 128;       // bytes of 64 elements of every slot
    static constexpr int TILE = PLANES * PLANE;         // K or V of a step
    static constexpr int P_BYTES = PLANE;               // one of the two 16-bit parts
    static constexpr int Q_PLANE = N * 128, Q_BYTES = PLANES * Q_PLANE;
    static constexpr int SMALL = (4 * N + 4 * N + 3 * N) * 4;  // warps' maxima and sums, m, sub, factor
    static constexpr int FIXED = 2 * P_BYTES + Q_BYTES + SMALL;
    static constexpr int MOST = 232448 - 2048;          // a CTA's shared memory, less the static part and the alignment
    static constexpr int FIT = (MOST - FIXED) / TILE;   // tiles; K's ring gets the odd one
    static constexpr int VS = FIT / 2 < 4 ? FIT / 2 : 4, KS = FIT - VS < 4 ? FIT - VS : 4;
    static_assert(VS >= 2, "the rings need two tiles each");
    // V is read as two planes whatever D is: behind the last one lies P
    static constexpr int SMEM = 1024 + (KS + VS) * TILE + FIXED;
    static constexpr int TMEM = N <= 16 ? 64 : N <= 32 ? 128 : 256;  // S, S, O of N columns each
};

// Byte of chunk c of row r in a plane.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
// Descriptor of an operand with the 128-byte swizzle (layout 2): `lbo` bytes
// from plane to plane (M-major), 1024 from eight rows to the next eight.
__device__ __forceinline__ uint64_t desc_swizzled(uint32_t at, uint32_t lbo) {
    return ((at >> 4) & 0x3FFFull) | (static_cast<uint64_t>(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// Instruction descriptor of kind::f16: fp32 accumulators, operands of type T.
template <typename T> constexpr uint32_t idesc_f16(int M, int N, bool a_major_m, bool b_major_n) {
    const uint32_t fmt = Half16<T>::type == ABRA_GGML_F16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((a_major_m ? 1u : 0u) << 15) | ((b_major_n ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
// This thread's TMEM lane, 16 columns.
__device__ __forceinline__ void tmem_ld16(uint32_t at, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
        "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// This thread's arrival at the barrier when its copies so far have landed.
__device__ __forceinline__ void copy_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Whether a phase has completed, without waiting for it.
__device__ __forceinline__ bool mbar_passed(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Barrier of the compute warps; true for all if `x` is for one of them.
template <int THREADS> __device__ __forceinline__ bool compute_any(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.aligned.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(x ? 1u : 0u), "n"(THREADS)
        : "memory");
    return r != 0;
}

// Folds v[0 .. N) over the warp's lanes with op; lane l ends with elements l *
// N / 32 .. (N >= 32), or element l / 2 (N = 16), in v[0 .. max(1, N / 32)).
template <int N, typename Op> __device__ __forceinline__ void fold_lanes(float (&v)[N], Op op) {
    const int lane = threadIdx.x & 31;
    int width = N;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        if (width > 1) {
            width >>= 1;
            const bool up = lane & d;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < width) {
                    const float give = up ? v[i] : v[i + width], keep = up ? v[i + width] : v[i];
                    v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, d));
                }
        } else {
            v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], d));
        }
    }
}
// Where fold_lanes leaves element e of lane l.
template <int N> __device__ __forceinline__ int folded(int lane, int e) { return N >= 32 ? lane * (N / 32) + e : lane >> 1; }

// Puts the infinities and NaNs that each row sees into its results (look_through),
// in tensor memory at `at`; all compute warps.  `codes`: [N][D], the place of the
// weights, which are at rest between two rows.
template <typename T, int D, int N>
__device__ __noinline__ void correct_results(const AttendArgs &p, int seq, int head, int from, int to, int all_see, int r0, uint32_t at,
                                             uint32_t *codes) {
    using S = Wide<D, N>;
    static_assert(N * D / 4 <= 2 * S::P_BYTES, "the codes fit the weights' place");
    const int tid = threadIdx.x, st = tid & 127, n_first = (tid >> 7) * S::NH;
    for (int i = tid; i < N * D / 16; i += S::COMPUTE) codes[i] = 0;
    named_bar_sync(1, S::COMPUTE);
    look_through<T, D, S::COMPUTE>(p, seq, head, from, to, all_see, r0, min(N, p.rows - r0), tid, codes);
    named_bar_sync(1, S::COMPUTE);
#pragma unroll 1
    for (int n0 = 0; n0 < S::NH; n0 += 16) {
        float o[16];
        tmem_ld16(at + n0, o);
        tmem_wait_ld();
        if (st < D) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = with_saw(o[i], codes, (n_first + n0 + i) * D + st);
        }
        __syncwarp();
        tmem_st16(at + n0, o);
    }
    tmem_wait_st();
}

template <typename T, int D, int N, bool SCORES>
__global__ void __launch_bounds__(Wide<D, N>::THREADS, 1) attend_wide_kernel(const __grid_constant__ AttendArgs p) {
    using S = Wide<D, N>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    __shared__ __align__(8) uint64_t k_full[S::KS], k_empty[S::KS], v_full[S::VS], v_empty[S::VS], s_done[2], o_done, q_ready, p_ready;
    __shared__ uint32_t s_tmem;
    unsigned char *s_k = smem, *s_v = smem + S::KS * S::TILE;  // rings
    unsigned char *s_p = s_v + S::VS * S::TILE, *s_q = s_p + 2 * S::P_BYTES;
    float *w_max = reinterpret_cast<float *>(s_q + S::Q_BYTES), *w_sum = w_max + 4 * N;  // [warp][N]
    float *s_m = w_sum + 4 * N, *s_sub = s_m + N, *s_fac = s_sub + N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    pdl_wait();
    pdl_launch_dependents();  // the join may take its place; it waits for the whole grid
    Walk<WIDE_STEP> w;
    Line line(0, 0);
    if (!find_start<S::THREADS>(p.kv, p.row_blocks, blockIdx.x, gridDim.x, p.resident, line, w)) return;
    const int begin = w.pos;
    if (tid == 0) {
        for (int i = 0; i < S::KS; ++i) mbar_init(&k_full[i], W_LOAD), mbar_init(&k_empty[i], 1);
        for (int i = 0; i < S::VS; ++i) mbar_init(&v_full[i], W_LOAD), mbar_init(&v_empty[i], 1);
        mbar_init(&q_ready, S::COMPUTE);
        mbar_init(&p_ready, S::COMPUTE);
        mbar_init(&s_done[0], 1);
        mbar_init(&s_done[1], 1);
        mbar_init(&o_done, 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(&s_tmem, S::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // after a wait that gave up (its error bit is set) nothing waits any more and
    // every loop runs to its end
    bool lost = false;
    auto wait = [&](uint64_t *bar, int parity) {
        if (!lost && !mbar_wait(bar, parity)) lost = true;
    };

    if (warp >= S::CW && warp < S::CW + 3) {
        // ---- loaders: eight rows of a step at a time, dealt to the three warps; a
        // lane answers for rows 8 (lw + 3 (l / 8)) + l % 8 and, l < 16, those of
        // the two groups after the warp's fourth ----
        constexpr int GROUPS = WIDE_STEP / 8, COPIES = S::CHUNKS / 4;  // of a lane for a group
        const int lw = warp - S::CW;
        int j = 0;
        do {
            for (int t0 = w.s.tile0 * WIDE_STEP; t0 < w.s.slot_end; t0 += WIDE_STEP, ++j) {
                int64_t off[2][2];  // K, V
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int t = t0 + 8 * (lw + 3 * (4 * y + (lane >> 3))) + (lane & 7);
                    int page = 0, in = 0;
                    if (t < min(w.s.slot_end, t0 + WIDE_STEP)) {
                        const int e = p.kv.page.div(t);
                        in = t - e * p.kv.a.page_size;
                        page = max(0, paged_page(p.kv, w.s.seq, e));
                    }
                    off[0][y] = paged_k_at(p.kv, page, w.s.head, in);
                    off[1][y] = paged_v_at(p.kv, page, w.s.head, in);
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    const int stages = kv ? S::VS : S::KS, st = j % stages;
                    if (j >= stages) wait(kv ? &v_empty[st] : &k_empty[st], (j / stages - 1) & 1);
                    const uint32_t to = smem_u32(kv ? s_v : s_k) + st * S::TILE;
                    const T *pool = static_cast<const T *>(kv ? p.kv.a.v : p.kv.a.k);
#pragma unroll
                    for (int q = 0; q < (GROUPS + 2) / 3; ++q) {
                        const int group = lw + 3 * q;
                        if (group >= GROUPS) break;
#pragma unroll
                        for (int i = 0; i < COPIES; ++i) {
                            const int x = 32 * i + lane, r = x / S::CHUNKS, chunk = x - r * S::CHUNKS, row = 8 * group + r;
                            const T *src = pool + __shfl_sync(0xffffffffu, off[kv][q / 4], 8 * (q % 4) + r) + 8 * chunk;
                            copy_async(to + (chunk >> 3) * S::PLANE + swizzled(row, chunk & 7), src, t0 + row < w.s.slot_end ? 16 : 0);
                        }
                    }
                    copy_arrive(kv ? &v_full[st] : &k_full[st]);
                }
            }
        } while (w.next(p.kv));
        copy_commit();
        copy_wait<0>();
    } else if (warp == S::CW + 3) {
        // ---- the tensor core's warp: all lanes run, one issues ----
        const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0), u_o = tmem + 2 * N;
        const uint32_t u_k = __shfl_sync(0xffffffffu, smem_u32(s_k), 0), u_v = __shfl_sync(0xffffffffu, smem_u32(s_v), 0);
        const uint32_t u_p = __shfl_sync(0xffffffffu, smem_u32(s_p), 0), u_q = __shfl_sync(0xffffffffu, smem_u32(s_q), 0);
        const bool leader = elect_one();
        auto issue_scores = [&](int it) {
            fence_proxy_async_smem();  // the loaders' copies, seen through the barrier, before the tensor core's reads
            tc_fence_after();
            const uint32_t k = __shfl_sync(0xffffffffu, u_k + it % S::KS * S::TILE, 0);
            const uint32_t d = __shfl_sync(0xffffffffu, tmem + (it & 1) * N, 0);
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    tc_mma_f16(d, desc_swizzled(k + ks / 4 * S::PLANE + ks % 4 * 32, 16),
                               desc_swizzled(u_q + ks / 4 * S::Q_PLANE + ks % 4 * 32, 16), idesc_f16<T>(128, N, false, false), ks > 0);
                tc_commit(&k_empty[it % S::KS]);
                tc_commit(&s_done[it & 1]);
            }
            __syncwarp();
        };
        auto issue_sum = [&](int it, bool first) {
            wait(&v_full[it % S::VS], (it / S::VS) & 1);
            fence_proxy_async_smem();
            tc_fence_after();
            const uint32_t v = __shfl_sync(0xffffffffu, u_v + it % S::VS * S::TILE, 0);
            if (leader) {
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int ks = 0; ks < WIDE_STEP / 16; ++ks)
                        tc_mma_f16(u_o, desc_swizzled(v + ks * 2048, S::PLANE), desc_swizzled(u_p + part * S::P_BYTES + ks * 2048, S::PLANE),
                                   idesc_f16<T>(128, N, true, true), part > 0 || ks > 0 ? 1u : !first);
                tc_commit(&v_empty[it % S::VS]);
                tc_commit(&o_done);
            }
            __syncwarp();
        };
        int it = 0, row = 0;
        do {
            const int n = (w.s.slot_end - w.s.tile0 * WIDE_STEP + WIDE_STEP - 1) / WIDE_STEP;
            wait(&q_ready, row++ & 1);
            wait(&k_full[it % S::KS], (it / S::KS) & 1);
            issue_scores(it);
            for (int k = 0; k < n; ++k, ++it) {
                // the next step's scores as soon as its keys have landed, this step's
                // sum as soon as its weights are there
                bool ahead = k + 1 == n;
                const uint64_t began = globaltimer_ns();
                while (!__all_sync(0xffffffffu, lost || mbar_passed(&p_ready, it & 1))) {
                    if (!ahead && __all_sync(0xffffffffu, lost || mbar_passed(&k_full[(it + 1) % S::KS], ((it + 1) / S::KS) & 1))) {
                        issue_scores(it + 1);
                        ahead = true;
                    }
                    if (globaltimer_ns() - began > WAIT_LIMIT_NS) {
                        report_error(ERR_WAIT_TIMEOUT);
                        lost = true;
                    }
                    lost = __any_sync(0xffffffffu, lost);
                }
                issue_sum(it, k == 0);
                if (!ahead) {
                    wait(&k_full[(it + 1) % S::KS], ((it + 1) / S::KS) & 1);
                    issue_scores(it + 1);
                }
            }
        } while (w.next(p.kv));
    } else {
        // ---- compute warps: thread t is slot t % 128 of a step and element t %
        // 128 of the results, for rows n_first .. n_first + NH - 1 ----
        constexpr int NH = S::NH;
        const int quarter = warp & 3, st = tid & 127, n_first = (tid >> 7) * NH;
        const uint32_t mine = s_tmem + (static_cast<uint32_t>(32 * quarter) << 16) + n_first, t_o = 2 * N;
        int it = 0;  // steps of this CTA so far
        do {
            const Segment &sg = w.s;
            const int r0 = sg.block * N, head = sg.head;
            // Q as an operand: rows past the end are zeros
            constexpr int QX = (N * S::CHUNKS + S::COMPUTE - 1) / S::COMPUTE;
            uint4 q[QX];
#pragma unroll
            for (int i = 0; i < QX; ++i) {
                const int x = i * S::COMPUTE + tid, r = x / S::CHUNKS, chunk = x - r * S::CHUNKS, row = r0 + r;
                q[i] = make_uint4(0, 0, 0, 0);
                if (r < N && row < p.rows) {
                    const int j = row / p.group, h = head * p.group + row - j * p.group;
                    q[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + (static_cast<int64_t>(sg.seq) * p.n_q + j) * p.ldq +
                                                            static_cast<int64_t>(h) * D + 8 * chunk);
                }
            }
#pragma unroll
            for (int i = 0; i < QX; ++i) {
                const int x = i * S::COMPUTE + tid, r = x / S::CHUNKS, chunk = x - r * S::CHUNKS;
                if (r < N) *reinterpret_cast<uint4 *>(s_q + (chunk >> 3) * S::Q_PLANE + swizzled(r, chunk & 7)) = q[i];
            }
            if (tid < N) s_m[tid] = -INFINITY, s_sub[tid] = 0.0f;
            fence_proxy_async_smem();
            mbar_arrive(&q_ready);
            named_bar_sync(1, S::COMPUTE);
            const int all_see = sg.len - p.n_q + 1;  // slots below are seen by every row
            float l[NH];
#pragma unroll
            for (int n = 0; n < NH; ++n) l[n] = 0.0f;
            bool odd = false;  // an infinity or NaN was taken out of a step
            const int j0 = (r0 + n_first) / p.group, rem0 = r0 + n_first - j0 * p.group;  // query of this thread's first row, head in the group
            for (int t0 = sg.tile0 * WIDE_STEP; t0 < sg.slot_end; t0 += WIDE_STEP, ++it) {
                const bool first = t0 == sg.tile0 * WIDE_STEP, edge = t0 + WIDE_STEP > all_see;
                const int t = t0 + st;
                // ---- scores in log2 units, masked; is a maximum to be raised? ----
                wait(&s_done[it & 1], (it >> 1) & 1);
                tc_fence_after();
                float s[NH];
                bool raise = false;
#pragma unroll
                for (int n0 = 0; n0 < NH; n0 += 16) tmem_ld16(mine + (it & 1) * N + n0, *reinterpret_cast<float (*)[16]>(s + n0));
                tmem_wait_ld();
#pragma unroll
                for (int n = 0; n < NH; ++n) s[n] *= p.scale_log2;
                if (edge) {
                    int j = j0, rem = rem0;
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        if (t >= min(sg.slot_end, all_see + min(j, p.n_q - 1))) s[n] = -INFINITY;
                        if (++rem == p.group) rem = 0, ++j;
                    }
                }
#pragma unroll
                for (int n0 = 0; n0 < NH; n0 += 4) {
                    const float4 m = *reinterpret_cast<const float4 *>(s_m + n_first + n0);
                    raise |= s[n0] - m.x > Weigh<T>::RAISE || s[n0 + 1] - m.y > Weigh<T>::RAISE || s[n0 + 2] - m.z > Weigh<T>::RAISE ||
                             s[n0 + 3] - m.w > Weigh<T>::RAISE;
                }
                if (SCORES && t < sg.slot_end) {
                    const int e = p.kv.page.div(t), page = paged_page(p.kv, sg.seq, e);
                    if (page >= 0) {  // a page outside the pool has no place for them
                        const int64_t at = score_at(p, sg.seq, head, t, paged_meta_at(p.kv, page, head, t - e * p.kv.a.page_size));
                        float *to = p.scores + at * (p.row_blocks * N) + r0 + n_first;
#pragma unroll
                        for (int n = 0; n < NH; n += 4) *reinterpret_cast<float4 *>(to + n) = make_float4(s[n], s[n + 1], s[n + 2], s[n + 3]);
                    }
                }
                raise = compute_any<S::COMPUTE>(raise);
                if (it > 0) wait(&o_done, (it - 1) & 1);  // the weights' buffer and the results are at rest
                tc_fence_after();
                if (raise) {
                    float top[NH];
#pragma unroll
                    for (int n = 0; n < NH; ++n) top[n] = s[n];
                    fold_lanes<NH>(top, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
                    for (int e = 0; e < (NH >= 32 ? NH / 32 : 1); ++e) w_max[quarter * N + n_first + folded<NH>(lane, e)] = top[e];
                    named_bar_sync(1, S::COMPUTE);
                    if (tid < N) {
                        const float m = s_m[tid];
                        const float now = fmaxf(fmaxf(fmaxf(w_max[tid], w_max[N + tid]), fmaxf(w_max[2 * N + tid], w_max[3 * N + tid])), m);
                        s_fac[tid] = scaled(m, now);
                        s_m[tid] = now;
                        s_sub[tid] = now == -INFINITY ? 0.0f : now;
                    }
                    named_bar_sync(1, S::COMPUTE);
                    if (!first) {
#pragma unroll
                        for (int n0 = 0; n0 < NH; n0 += 16) {
                            float o[16];
                            tmem_ld16(mine + t_o + n0, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                o[i] *= s_fac[n_first + n0 + i];
                                l[n0 + i] *= s_fac[n_first + n0 + i];
                            }
                            tmem_st16(mine + t_o + n0, o);
                        }
                        tmem_wait_st();
                    }
                }
                if (edge && p.n_q > 1 && n_first == 0) {  // not every row sees them all: look_through
                    wait(&v_full[it % S::VS], (it / S::VS) & 1);
                    for (int c = 0; c < S::CHUNKS; ++c) {
                        uint4 *v = reinterpret_cast<uint4 *>(s_v + it % S::VS * S::TILE + (c >> 3) * S::PLANE +
                                                             swizzled(st, c & 7));
                        bool any = false;
                        const uint4 x = make_uint4(finite_part<T>(v->x, any), finite_part<T>(v->y, any), finite_part<T>(v->z, any),
                                                   finite_part<T>(v->w, any));
                        if (any) *v = x, odd = true;
                    }
                }
                // ---- weights, as the sum of two 16-bit values (one rounding would
                // cost as much precision as the result's own) ----
#pragma unroll
                for (int n0 = 0; n0 < NH; n0 += 8) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const int n = n0 + i;
                        const float2 sub = *reinterpret_cast<const float2 *>(s_sub + n_first + n);
                        const float a = weight_of<T>(s[n], sub.x), b = weight_of<T>(s[n + 1], sub.y);
                        l[n] += a;
                        l[n + 1] += b;
                        hi[i / 2] = pack2<T>(a, b);
                        const float2 h = unpack2<T>(hi[i / 2]);
                        lo[i / 2] = pack2<T>(a - h.x, b - h.y);
                    }
                    unsigned char *to = s_p + swizzled(st, (n_first + n0) / 8);
                    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(to + S::P_BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                tc_fence_before();
                fence_proxy_async_smem();
                mbar_arrive(&p_ready);
            }

            // ---- the row's end ----
            fold_lanes<NH>(l, [](float a, float b) { return a + b; });
#pragma unroll
            for (int e = 0; e < (NH >= 32 ? NH / 32 : 1); ++e) w_sum[quarter * N + n_first + folded<NH>(lane, e)] = l[e];
            odd = compute_any<S::COMPUTE>(odd);
            const bool whole = sg.tile0 == 0 && sg.tile1 == sg.n;
            const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (w.pos == begin ? 0 : 1);
            if (tid < N && r0 + tid < p.rows) {
                const float total = w_sum[tid] + w_sum[N + tid] + w_sum[2 * N + tid] + w_sum[3 * N + tid];
                if (whole) finish_lse<T>(p, sg.seq, head, r0 + tid, s_m[tid], total);
                else p.part_ml[slot * N + tid] = make_float2(s_m[tid], total);
                s_fac[tid] = total != 0.0f ? 1.0f / total : 0.0f;
            }
            named_bar_sync(1, S::COMPUTE);
            wait(&o_done, (it - 1) & 1);
            tc_fence_after();
            if (sg.tile0 == 0 && tid == 0)
                p.split[static_cast<int64_t>(sg.seq) * w.units + sg.unit] =
                    make_int2(static_cast<int>(slot), whole ? static_cast<int>(blockIdx.x) : line.piece(sg.row_begin + ROW_COST + sg.n - 1));
            auto look = [&]() {
                correct_results<T, D, N>(p, sg.seq, head, sg.tile0 * WIDE_STEP, sg.slot_end, all_see, r0, mine + t_o, reinterpret_cast<uint32_t *>(s_p));
            };
            if (odd) look();
            for (;;) {
                bool unexplained = false;  // a NaN of a row whose weights have none
#pragma unroll 1
                for (int n0 = 0; n0 < NH; n0 += 16) {
                    const int n = n_first + n0, nr = min(16, p.rows - r0 - n);
                    float o[16];
                    tmem_ld16(mine + t_o + n0, o);
                    tmem_wait_ld();
                    if (st >= D || nr <= 0) continue;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[i % 4] += o[i];
                    if (isnan((sum[0] + sum[1]) + (sum[2] + sum[3]))) {
#pragma unroll 1
                        for (int i = 0; i < nr; ++i) unexplained |= !isnan(s_fac[n + i]);
                    }
                    if (!whole) {
                        float *to = p.part_o + (slot * N + n) * D + st;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (i < nr) to[i * D] = o[i];
                    } else {
                        int j = (r0 + n) / p.group, rem = r0 + n - j * p.group;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int64_t to = (static_cast<int64_t>(sg.seq) * p.n_q + j) * p.ldo + static_cast<int64_t>(head * p.group + rem) * D + st;
                            const float x = s_fac[n + i] != 0.0f ? o[i] * s_fac[n + i] : 0.0f;
                            if (i < nr) {
                                if (p.out_f32) static_cast<float *>(p.out)[to] = x;
                                else static_cast<T *>(p.out)[to] = Half16<T>::down(x);
                            }
                            if (++rem == p.group) rem = 0, ++j;
                        }
                    }
                }
                tc_fence_before();
                // Q, the sums and the results are free again, or are stored once more
                if (!compute_any<S::COMPUTE>(!odd && unexplained)) break;
                tc_fence_after();
                odd = true;
                look();
            }
        } while (w.next(p.kv));
    }
    __syncthreads();
    if (warp == 0) tmem_dealloc(s_tmem, S::TMEM);
}

template <typename T, int D, int N, bool SCORES> cudaError_t launch_one(const AttendArgs &p, int pieces, cudaStream_t st) {
    constexpr int smem = Wide<D, N>::SMEM;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = paged_smem(reinterpret_cast<const void *>(attend_wide_kernel<T, D, N, SCORES>), smem, done);
    if (e != cudaSuccess) return e;
    return paged_launch(attend_wide_kernel<T, D, N, SCORES>, dim3(pieces), Wide<D, N>::THREADS, smem, st, p);
}
template <typename T, int D, int N> cudaError_t launch_scores(const AttendArgs &p, int pieces, bool scores, cudaStream_t st) {
    return scores ? launch_one<T, D, N, true>(p, pieces, st) : launch_one<T, D, N, false>(p, pieces, st);
}
template <typename T, int D> cudaError_t launch_rows(const AttendArgs &p, int n, int pieces, bool scores, cudaStream_t st) {
    return n == 16   ? launch_scores<T, D, 16>(p, pieces, scores, st)
           : n == 32 ? launch_scores<T, D, 32>(p, pieces, scores, st)
                     : launch_scores<T, D, 64>(p, pieces, scores, st);
}
template <typename T> cudaError_t launch_dim(const AttendArgs &p, int n, int pieces, bool scores, cudaStream_t st) {
    switch (p.kv.a.head_dim) {
        case 64: return launch_rows<T, 64>(p, n, pieces, scores, st);
        case 96: return launch_rows<T, 96>(p, n, pieces, scores, st);
        default: return launch_rows<T, 128>(p, n, pieces, scores, st);
    }
}

}  // namespace

cudaError_t launch_attend_wide(const AttendArgs &p, int n, int pieces, bool scores, cudaStream_t st) {
    return p.kv.a.type == ABRA_GGML_F16 ? launch_dim<__half>(p, n, pieces, scores, st)
                                        : launch_dim<__nv_bfloat16>(p, n, pieces, scores, st);
}

}  // namespace abra

ABRA_ERROR_WORD_ACCESSOR(paged_attention_wide_error_word)
