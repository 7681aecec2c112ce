// paged_attention.cu -- attention of each sequence's newest tokens over its
// paged key-value cache, with the slots' accumulated weights
// (abra_paged_attention).
//
// For query j of n_q, q head h of kv head g: s_t = scale q.k_t over the slots t
// < len - (n_q - 1 - j), lse = log sum_t exp s_t, out = sum_t exp(s_t - lse)
// v_t; acc_t += exp(s_t - lse) over the group's heads and the n_q queries.
//
// Bound: a slot of one kv head is 4 D bytes for 4 D flops a row, and a kv head
// has few rows (group x n_q), so the kernel is bound by reading the cache once.
// The work is cut evenly whatever the lengths are: the steps of 64 slots of all
// (sequence, kv head, block of rows) triples form one line, and each of the
// resident CTAs takes an equal piece of it, crossing from triple to triple.
//
// Layout: both products run on the tensor cores with the slots (16 a warp) as
// the tall side and the rows (8 a tile) as the narrow one, S^T = K Q^T and O^T
// = V^T P^T, so that a group of four heads wastes half a tile and not three
// quarters.  No shared memory: the order of the contracted index is free as
// long as both operands agree, so lane (g, c) = (lane / 4, lane % 4) reads 16
// contiguous bytes of K rows g and g + 8 (elements 32 i + 8 c ..) and takes
// them as the A fragments of two k-steps, with Q read the same way; of V it
// reads rows 2c, 2c+1, 2c+8, 2c+9 (elements 64 j + 8 g ..) and pairs slots
// with byte permutes.  Each lane's next K tile is in flight while this tile's
// softmax runs, and its next V tile during the next scores.
#include "paged_kv.cuh"

namespace abra {
namespace {

constexpr int AT_WARPS = 4, AT_THREADS = AT_WARPS * 32;
constexpr int TILE = 16;                  // slots of a warp's tile
constexpr int STEP = TILE * AT_WARPS;     // slots of a CTA's step
constexpr int SCAN = AT_THREADS;          // sequences of one block scan
// A row's maximum is raised only when a score passes it by 2^RAISE: weights
// stay below 2^RAISE (well inside fp16), and most tiles need no reduction.
constexpr float RAISE = 10.0f;
constexpr int MAX_CTAS = 4;  // a multiprocessor

struct AttendArgs {
    PagedKv kv;
    const void *q;
    void *out;
    float *lse;
    int64_t ldq, ldo;
    float scale_log2;  // scale / ln 2: scores are kept in units of log2
    int n_heads, n_q, group, rows, row_blocks, out_f32;
    // workspace
    unsigned *arrived;  // [cta] segments done of the split row that begins in that CTA's piece (at most one)
    float *part_o;      // [cta][2][8 NT][D]
    float2 *part_ml;    // [cta][2][8 NT] maximum (log2 units) and sum
    float *row_lse;     // [seq][kv head][row] log2 of the sum, +inf for a row that sees nothing
    float *scores;      // [page][kv head][offset][padded rows], log2 units
};

// ------------------------------------------------------------------ PTX ---
__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 x;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "l"(p));
    return x;
}
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                    uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                           uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 matrix of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t x);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&x));
}
// The packed pair with its infinities and NaNs as zeros; `any` collects them.
template <typename T> __device__ __forceinline__ uint32_t finite_part(uint32_t x, bool &any) {
    constexpr uint32_t EXP = Half16<T>::type == ABRA_GGML_F16 ? 0x7c00u : 0x7f80u;
    if ((x & EXP) == EXP) x &= 0xffff0000u, any = true;
    if ((x & (EXP << 16)) == (EXP << 16)) x &= 0x0000ffffu, any = true;
    return x;
}

// ------------------------------------------------------------ the line ---
// Where CTA `cta` of `ctas` starts on the line of steps.
struct Line {
    int64_t total;  // steps of all triples
    int ctas;       // pieces; each has at least one step
    __device__ __forceinline__ int64_t begin(int cta) const { return cta * total / ctas; }
    // the piece that holds step x
    __device__ __forceinline__ int piece(int64_t x) const { return static_cast<int>(((x + 1) * ctas - 1) / total); }
};
__device__ __forceinline__ int steps_of(int len) { return (len + STEP - 1) / STEP; }

struct Start {
    int seq;        // the sequence of the piece's first step
    int64_t steps;  // steps of the sequences before it (for one unit)
};

// Sums the sequences' steps and finds the one that this CTA's piece begins in.
// `units` triples share a sequence's length.  All threads of the block.
__device__ __forceinline__ Line find_start(const PagedKv &kv, int units, Start &at) {
    __shared__ unsigned s_warp[AT_WARPS];
    __shared__ int s_seq;
    __shared__ int64_t s_steps;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = kv.a.n_seqs;
    // inclusive scan of the steps of sequences base .. base + SCAN - 1
    unsigned own = 0, incl = 0, all = 0;
    auto scan = [&](int base) {
        own = base + tid < n ? static_cast<unsigned>(steps_of(paged_len(kv, base + tid))) : 0u;
        incl = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += y;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int w = 0; w < AT_WARPS; ++w) {
            if (w < warp) incl += s_warp[w];
            all += s_warp[w];
        }
    };
    int64_t sum = 0;
    int base = 0;
    for (; base < n; base += SCAN) {
        scan(base);
        sum += all;
    }
    Line line{sum * units, 0};
    line.ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), line.total));
    if (static_cast<int>(blockIdx.x) >= line.ctas) return line;
    const int64_t x = line.begin(blockIdx.x) / units;
    int64_t before = 0;
    if (n <= SCAN) {
        if (incl > x && incl - own <= x) s_seq = tid, s_steps = incl - own;
    } else {
        for (base = 0; base < n; base += SCAN) {
            scan(base);
            if (before + incl > x && before + incl - own <= x) s_seq = base + tid, s_steps = before + incl - own;
            before += all;
            if (before > x) break;
        }
    }
    __syncthreads();
    at = {s_seq, s_steps};
    return line;
}

// --------------------------------------------------------------- kernel ---
template <int D, int NT> struct Shape {
    static constexpr int NK = D / 32;           // 16-byte pieces of a K row a lane reads
    static constexpr int NV = (D + 63) / 64;    // 16-byte pieces of a V row a lane reads
    static constexpr int MT = NV * 4;           // 16-element tiles of the output
    static constexpr int R = 8 * NT;            // rows of a block
    static constexpr int PITCH = D + 4;         // floats of a row in the join buffer
    static constexpr int MIN_CTAS = NT == 1 ? 3 : 2;
    static constexpr int Q_BYTES = NT == 1 ? 0 : NT * NK * 32 * 16;
    static constexpr int SMEM = Q_BYTES + AT_WARPS * R * (PITCH + 2) * 4;
};

template <typename T>
__device__ __forceinline__ void store_out(const AttendArgs &p, int64_t at, float4 x) {
    if (p.out_f32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = x;
    } else {
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    }
}

// A finished row: out at elements d .. d + 3 (lanes of one warp share the
// row), its lse by the lane of element 0.  total == 0: the row saw nothing.
template <typename T>
__device__ __forceinline__ void finish_row(const AttendArgs &p, int seq, int head, int r, int d, int D, float4 o, float m,
                                           float total) {
    const int j = r / p.group, h = head * p.group + r - j * p.group;
    const int64_t row = static_cast<int64_t>(seq) * p.n_q + j;
    const float inv = total != 0.0f ? 1.0f / total : 0.0f;
    store_out<T>(p, row * p.ldo + static_cast<int64_t>(h) * D + d,
                 total != 0.0f ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0, 0, 0, 0));
    if (d == 0) {
        const float l2 = total != 0.0f ? m + log2f(total) : -INFINITY;
        if (p.lse) p.lse[row * p.n_heads + h] = l2 * 0.69314718055994531f;
        if (p.row_lse)
            p.row_lse[(static_cast<int64_t>(seq) * p.kv.a.n_kv_heads + head) * p.rows + r] = total != 0.0f ? l2 : INFINITY;
    }
}

template <typename T, int D, int NT, bool SCORES>
__global__ void __launch_bounds__(AT_THREADS, Shape<D, NT>::MIN_CTAS) attend_kernel(const __grid_constant__ AttendArgs p) {
    using S = Shape<D, NT>;
    extern __shared__ __align__(16) unsigned char smem[];
    uint4 *s_q = reinterpret_cast<uint4 *>(smem);  // [NT][NK][32 lanes] Q fragments (NT > 1)
    float *s_o = reinterpret_cast<float *>(smem + S::Q_BYTES);  // [warp][R][PITCH]
    float *s_m = s_o + AT_WARPS * S::R * S::PITCH, *s_l = s_m + AT_WARPS * S::R;
    __shared__ bool s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int units = p.kv.a.n_kv_heads * p.row_blocks;
    const T *kp = static_cast<const T *>(p.kv.a.k), *vp = static_cast<const T *>(p.kv.a.v);

    Start at;
    const Line line = find_start(p.kv, units, at);
    // rows of empty sequences are nobody's: zeros and -infinity
    for (int s = blockIdx.x; s < p.kv.a.n_seqs; s += gridDim.x) {
        if (paged_len(p.kv, s) > 0) continue;
        for (int i = tid; i < p.kv.a.n_kv_heads * p.rows * (D / 4); i += AT_THREADS) {
            const int row = i / (D / 4), head = row / p.rows;
            finish_row<T>(p, s, head, row - head * p.rows, (i - row * (D / 4)) * 4, D, make_float4(0, 0, 0, 0), 0.0f, 0.0f);
        }
    }
    if (static_cast<int>(blockIdx.x) >= line.ctas) return;

    int64_t pos = line.begin(blockIdx.x);
    const int64_t begin = pos, end = line.begin(blockIdx.x + 1);
    int seq = at.seq;
    int64_t seq_begin = at.steps * units;
    int len = paged_len(p.kv, seq);
    while (pos < end) {
        // the segment: steps [tile0, tile1) of row block u of this sequence
        const int n = steps_of(len);
        const int u = static_cast<int>((pos - seq_begin) / n);
        const int64_t row_begin = seq_begin + static_cast<int64_t>(u) * n;
        const int tile0 = static_cast<int>(pos - row_begin), tile1 = static_cast<int>(min(static_cast<int64_t>(n), end - row_begin));
        const int head = u / p.row_blocks, r0 = (u - head * p.row_blocks) * S::R;
        const int slot_end = min(len, tile1 * STEP);

        // Q fragments: row r0 + 8 nt + g, elements 32 i + 8 c ..; rows past the end are zeros
        uint4 qf[NT == 1 ? S::NK : 1];
        auto load_q = [&](int nt, int i) {
            const int r = r0 + 8 * nt + g;
            if (r >= p.rows) return make_uint4(0, 0, 0, 0);
            const int j = r / p.group, h = head * p.group + r - j * p.group;
            return __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + (static_cast<int64_t>(seq) * p.n_q + j) * p.ldq +
                                                         static_cast<int64_t>(h) * D + 32 * i + 8 * c));
        };
        if (NT == 1) {
#pragma unroll
            for (int i = 0; i < S::NK; ++i) qf[NT == 1 ? i : 0] = load_q(0, i);
        } else {
            for (int x = warp; x < NT * S::NK; x += AT_WARPS) s_q[x * 32 + lane] = load_q(x / S::NK, x % S::NK);
            __syncthreads();
        }
        // slots that rows 2c, 2c + 1 of each tile see
        int seen[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) seen[nt][e] = len - (p.n_q - 1 - min((r0 + 8 * nt + 2 * c + e) / p.group, p.n_q - 1));
        const int all_see = len - p.n_q + 1;  // slots below are seen by every row

        float o[NT][S::MT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int mt = 0; mt < S::MT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
        }

        // lane's row of a tile is slot base + lane % 16: its page, then its offsets
        const int64_t table_row = static_cast<int64_t>(seq) * p.kv.a.table_stride;
        auto fetch_page = [&](int base) {
            const int t = base + (lane & 15);
            return t < slot_end ? __ldg(p.kv.a.table + table_row + p.kv.page.div(t)) : 0;
        };
        int64_t k_off, v_off, meta_off;
        auto address = [&](int base, int page) {
            const int t = base + (lane & 15), off = t - p.kv.page.div(t) * p.kv.a.page_size;
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.kv.a.n_pages)) {
                report_error(ERR_BAD_INDEX);
                page = 0;
            }
            k_off = paged_k_at(p.kv, page, head, off);
            v_off = paged_v_at(p.kv, page, head, off);
            if (SCORES) meta_off = paged_meta_at(p.kv, page, head, off) * (p.row_blocks * S::R) + r0;
        };
        uint4 kf[2][S::NK], vf[4][S::NV];
        auto load_k = [&](int base) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int row = g + 8 * x;
                const T *src = kp + __shfl_sync(0xffffffffu, k_off, row) + 8 * c;
                const bool ok = base + row < slot_end;
#pragma unroll
                for (int i = 0; i < S::NK; ++i) kf[x][i] = ok ? ld_stream(src + 32 * i) : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_v = [&](int base, int64_t off) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = 2 * c + (x & 1) + 8 * (x >> 1);
                const T *src = vp + __shfl_sync(0xffffffffu, off, row) + 8 * g;
                const bool ok = base + row < slot_end;
#pragma unroll
                for (int j = 0; j < S::NV; ++j)
                    vf[x][j] = ok && 64 * j + 8 * g < D ? ld_stream(src + 64 * j) : make_uint4(0, 0, 0, 0);
            }
        };

        int base = tile0 * STEP + warp * TILE;
        if (base < slot_end) {
            address(base, fetch_page(base));
            load_k(base);
            load_v(base, v_off);
            int page_next = fetch_page(base + STEP);
            for (; base < slot_end; base += STEP) {
                // scores: rows of the tile (slots g, g + 8) by rows of the block (2c, 2c + 1)
                float sc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
                for (int i = 0; i < S::NK; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 q = NT == 1 ? qf[NT == 1 ? i : 0] : s_q[(nt * S::NK + i) * 32 + lane];
                        mma_16x8x16<T>(sc[nt], kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, q.x, q.y);
                        mma_16x8x16<T>(sc[nt], kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, q.z, q.w);
                    }
                const int64_t v_this = v_off, meta_this = meta_off;
                const int next = base + STEP;
                if (next < slot_end) {
                    address(next, page_next);
                    load_k(next);
                    page_next = fetch_page(next + STEP);
                }
                // log2 units, the mask, and the rows' maxima
                const bool edge = base + TILE > all_see;
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[nt][e] *= p.scale_log2;
                        if (edge && base + g + 8 * (e >> 1) >= min(seen[nt][e & 1], slot_end)) sc[nt][e] = -INFINITY;
                        raise |= sc[nt][e] > m[nt][e & 1] + RAISE;
                    }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(sc[nt][e], sc[nt][e + 2]);
#pragma unroll
                            for (int x = 4; x <= 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                            top = fmaxf(top, m[nt][e]);
                            const float f = top == m[nt][e] ? 1.0f : exp2_fast(m[nt][e] - top);
                            m[nt][e] = top;
                            l[nt][e] *= f;
#pragma unroll
                            for (int mt = 0; mt < S::MT; ++mt) o[nt][mt][e] *= f, o[nt][mt][e + 2] *= f;
                        }
                }
                if (SCORES) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int64_t to = __shfl_sync(0xffffffffu, meta_this, g + 8 * x);
                        if (base + g + 8 * x < slot_end)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                *reinterpret_cast<float2 *>(p.scores + to + 8 * nt + 2 * c) = make_float2(sc[nt][2 * x], sc[nt][2 * x + 1]);
                    }
                }
                // weights, as the sum of two 16-bit values: the tensor cores take
                // 16-bit operands, and one rounding would cost as much precision
                // as the result's own
                uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float mm = m[nt][e & 1];
                        sc[nt][e] = exp2_fast(sc[nt][e] - (mm == -INFINITY ? 0.0f : mm));
                        l[nt][e & 1] += sc[nt][e];
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t h = pack2<T>(sc[nt][2 * x], sc[nt][2 * x + 1]);
                        const float2 f = unpack2<T>(h);
                        hi[nt][x] = trans8x8(h);
                        lo[nt][x] = trans8x8(pack2<T>(sc[nt][2 * x] - f.x, sc[nt][2 * x + 1] - f.y));
                    }
                }
                // A slot that only some rows see has weight 0 in the others, and 0
                // times an infinity or NaN in its V row would reach them: such
                // elements are taken out here and added row by row below.
                bool odd = false;
                if (edge && p.n_q > 1) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int j = 0; j < S::NV; ++j) {
                            vf[x][j].x = finite_part<T>(vf[x][j].x, odd);
                            vf[x][j].y = finite_part<T>(vf[x][j].y, odd);
                            vf[x][j].z = finite_part<T>(vf[x][j].z, odd);
                            vf[x][j].w = finite_part<T>(vf[x][j].w, odd);
                        }
                    odd = __any_sync(0xffffffffu, odd);
                }
#pragma unroll
                for (int mt = 0; mt < S::MT; ++mt) {
                    const uint32_t v0 = reinterpret_cast<const uint32_t *>(&vf[0][mt / 4])[mt % 4];
                    const uint32_t v1 = reinterpret_cast<const uint32_t *>(&vf[1][mt / 4])[mt % 4];
                    const uint32_t v2 = reinterpret_cast<const uint32_t *>(&vf[2][mt / 4])[mt % 4];
                    const uint32_t v3 = reinterpret_cast<const uint32_t *>(&vf[3][mt / 4])[mt % 4];
                    const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
                    const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16x8x16<T>(o[nt][mt], a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
                        mma_16x8x16<T>(o[nt][mt], a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
                    }
                }
                if (odd) {
                    for (int t = 0; t < TILE; ++t) {
                        const T *src = vp + __shfl_sync(0xffffffffu, v_this, t) + 8 * g;
                        const int from = (t & 7) * 4 + c;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float w0 = __shfl_sync(0xffffffffu, t < 8 ? sc[nt][0] : sc[nt][2], from);
                            const float w1 = __shfl_sync(0xffffffffu, t < 8 ? sc[nt][1] : sc[nt][3], from);
                            if (base + t >= slot_end) continue;
#pragma unroll
                            for (int mt = 0; mt < S::MT; ++mt) {
                                if (64 * (mt / 4) + 8 * g >= D) continue;
                                const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t *>(src + 64 * (mt / 4) + 2 * (mt % 4)));
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float v = e ? f.y : f.x;
                                    if (isfinite(v)) continue;
                                    if (base + t < seen[nt][0]) o[nt][mt][2 * e] += w0 * v;
                                    if (base + t < seen[nt][1]) o[nt][mt][2 * e + 1] += w1 * v;
                                }
                            }
                        }
                    }
                }
                if (next < slot_end) load_v(next, v_off);
            }
        }

        // ---- join the warps: maximum, then scaled sums in shared memory ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
                if (g == 0) {
                    s_m[warp * S::R + 8 * nt + 2 * c + e] = m[nt][e];
                    s_l[warp * S::R + 8 * nt + 2 * c + e] = l[nt][e];
                }
            }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * nt + 2 * c + e;
                float top = s_m[r];
#pragma unroll
                for (int w = 1; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w * S::R + r]);
                const float f = m[nt][e] == top ? 1.0f : exp2_fast(m[nt][e] - top);
                float *dst = s_o + (warp * S::R + r) * S::PITCH;
#pragma unroll
                for (int mt = 0; mt < S::MT; mt += 2) {
                    const int d = 64 * (mt / 4) + 8 * g + 2 * (mt % 4);
                    if (d < D)
                        *reinterpret_cast<float4 *>(dst + d) = make_float4(o[nt][mt][e] * f, o[nt][mt][e + 2] * f,
                                                                           o[nt][mt + 1][e] * f, o[nt][mt + 1][e + 2] * f);
                }
            }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == n;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (pos == begin ? 0 : 1);
        for (int i = tid; i < S::R * (D / 4); i += AT_THREADS) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            if (r0 + r >= p.rows) break;
            float top = s_m[r], total = 0.0f;
#pragma unroll
            for (int w = 1; w < AT_WARPS; ++w) top = fmaxf(top, s_m[w * S::R + r]);
            float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < AT_WARPS; ++w) {
                const float mw = s_m[w * S::R + r];
                total += s_l[w * S::R + r] * (mw == top ? 1.0f : exp2_fast(mw - top));
                const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * S::R + r) * S::PITCH + d);
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
            }
            if (whole) {
                finish_row<T>(p, seq, head, r0 + r, d, D, sum, top, total);
            } else {
                *reinterpret_cast<float4 *>(p.part_o + (slot * S::R + r) * D + d) = sum;
                if (d == 0) p.part_ml[slot * S::R + r] = make_float2(top, total);
            }
        }
        if (!whole) {
            // ---- the last of the row's segments to arrive joins them, in order ----
            const int first = line.piece(row_begin), last = line.piece(row_begin + n - 1);
            unsigned *arrived = p.arrived + first;
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(arrived, 1u) == static_cast<unsigned>(last - first);
            __syncthreads();
            if (s_last) {
                __threadfence();
                if (tid == 0) *arrived = 0;  // ready for the next call
                for (int r = warp; r < S::R && r0 + r < p.rows; r += AT_WARPS) {
                    // piece x holds the row's segment in its first slot unless it begins before the row
                    auto slot_of = [&](int x) { return (static_cast<int64_t>(x) * 2 + (line.begin(x) < row_begin ? 1 : 0)) * S::R + r; };
                    float top = -INFINITY;
                    for (int x = first + lane; x <= last; x += 32) top = fmaxf(top, __ldcg(p.part_ml + slot_of(x)).x);
#pragma unroll
                    for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    float total = 0.0f;
                    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
                    for (int x = first; x <= last; ++x) {
                        const int64_t from = slot_of(x);
                        const float2 ml = __ldcg(p.part_ml + from);
                        const float f = ml.x == top ? 1.0f : exp2_fast(ml.x - top);
                        total += ml.y * f;
                        if (lane < D / 4) {
                            const float4 y = __ldcg(reinterpret_cast<const float4 *>(p.part_o + from * D + 4 * lane));
                            sum.x += f * y.x, sum.y += f * y.y, sum.z += f * y.z, sum.w += f * y.w;
                        }
                    }
                    if (lane < D / 4) finish_row<T>(p, seq, head, r0 + r, 4 * lane, D, sum, top, total);
                }
            }
        }
        __syncthreads();  // the join buffer and Q are free again
        pos = row_begin + tile1;
        if (pos < end && pos == seq_begin + static_cast<int64_t>(n) * units) {
            seq_begin = pos;
            do len = paged_len(p.kv, ++seq);
            while (len == 0);
        }
    }
}

// acc += the slots' weights: exp2(score - lse) summed over the rows, a thread
// for four rows of a slot, on the same line of steps as the attention.
template <int QUADS>  // float4s of a slot's padded rows that neighbouring lanes share
__global__ void __launch_bounds__(AT_THREADS) accumulate_kernel(const __grid_constant__ AttendArgs p, int padded) {
    const int tid = threadIdx.x, heads = p.kv.a.n_kv_heads;
    Start at;
    const Line line = find_start(p.kv, heads, at);
    if (static_cast<int>(blockIdx.x) >= line.ctas) return;
    int64_t pos = line.begin(blockIdx.x);
    const int64_t end = line.begin(blockIdx.x + 1);
    int seq = at.seq;
    int64_t seq_begin = at.steps * heads;
    int len = paged_len(p.kv, seq);
    const int part = tid % QUADS;
    while (pos < end) {
        const int n = steps_of(len);
        const int head = static_cast<int>((pos - seq_begin) / n);
        const int64_t row_begin = seq_begin + static_cast<int64_t>(head) * n;
        const int tile0 = static_cast<int>(pos - row_begin), tile1 = static_cast<int>(min(static_cast<int64_t>(n), end - row_begin));
        const int slot_end = min(len, tile1 * STEP);
        const float *lse = p.row_lse + (static_cast<int64_t>(seq) * heads + head) * p.rows;
        for (int t0 = tile0 * STEP; t0 < slot_end; t0 += AT_THREADS / QUADS) {
            const int t = t0 + tid / QUADS;
            float sum = 0.0f;
            int64_t meta = -1;
            if (t < slot_end) {
                const int e = p.kv.page.div(t), page = paged_page(p.kv, seq, e);
                if (page >= 0) {
                    meta = paged_meta_at(p.kv, page, head, t - e * p.kv.a.page_size);
                    for (int r = 4 * part; r < p.rows; r += 4 * QUADS) {
                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(p.scores + meta * padded + r));
                        sum += exp2_fast(x.x - __ldcg(lse + r));
                        if (r + 1 < p.rows) sum += exp2_fast(x.y - __ldcg(lse + r + 1));
                        if (r + 2 < p.rows) sum += exp2_fast(x.z - __ldcg(lse + r + 2));
                        if (r + 3 < p.rows) sum += exp2_fast(x.w - __ldcg(lse + r + 3));
                    }
                }
            }
#pragma unroll
            for (int x = 1; x < QUADS; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (meta >= 0 && part == 0) p.kv.a.acc[meta] += sum;
        }
        pos = row_begin + tile1;
        if (pos < end && pos == seq_begin + static_cast<int64_t>(n) * heads) {
            seq_begin = pos;
            do len = paged_len(p.kv, ++seq);
            while (len == 0);
        }
    }
}

// ------------------------------------------------------------------ host ---
struct Plan {
    int nt, row_blocks, ctas, sms;
    int64_t arrived, part_o, part_ml, row_lse, scores, bytes;  // workspace offsets
};

int tile_count(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

int make_plan(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q, bool accumulate, Plan &pl) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&pl.sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return paged_cuda(e, "device properties");
    const int rows = n_heads / kv->n_kv_heads * n_q;
    pl.nt = tile_count(rows);
    pl.row_blocks = (rows + 8 * pl.nt - 1) / (8 * pl.nt);
    pl.ctas = pl.sms * (pl.nt == 1 ? 3 : 2);
    const int64_t padded = static_cast<int64_t>(pl.row_blocks) * 8 * pl.nt;
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    int64_t at = 0;
    pl.arrived = at, at = up(at + static_cast<int64_t>(pl.sms) * MAX_CTAS * 4);  // the same place for all arguments
    pl.part_o = at, at = up(at + static_cast<int64_t>(pl.ctas) * 2 * 8 * pl.nt * kv->head_dim * 4);
    pl.part_ml = at, at = up(at + static_cast<int64_t>(pl.ctas) * 2 * 8 * pl.nt * 8);
    pl.row_lse = pl.scores = at;
    if (accumulate) {
        at = up(at + static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads * rows * 4);
        pl.scores = at;
        at = up(at + static_cast<int64_t>(kv->n_pages) * kv->n_kv_heads * kv->page_size * padded * 4);
    }
    pl.bytes = at + 256;
    return ABRA_OK;
}

template <typename T, int D, int NT, bool SCORES>
cudaError_t launch_one(const AttendArgs &p, const Plan &pl, cudaStream_t st) {
    constexpr int smem = Shape<D, NT>::SMEM;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, D, NT, SCORES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    attend_kernel<T, D, NT, SCORES><<<pl.ctas, AT_THREADS, smem, st>>>(p);
    return cudaGetLastError();
}
template <typename T, int D, bool SCORES>
cudaError_t launch_rows(const AttendArgs &p, const Plan &pl, cudaStream_t st) {
    return pl.nt == 1   ? launch_one<T, D, 1, SCORES>(p, pl, st)
           : pl.nt == 2 ? launch_one<T, D, 2, SCORES>(p, pl, st)
                        : launch_one<T, D, 4, SCORES>(p, pl, st);
}
template <typename T, bool SCORES> cudaError_t launch_dim(const AttendArgs &p, const Plan &pl, cudaStream_t st) {
    switch (p.kv.a.head_dim) {
        case 64: return launch_rows<T, 64, SCORES>(p, pl, st);
        case 96: return launch_rows<T, 96, SCORES>(p, pl, st);
        default: return launch_rows<T, 128, SCORES>(p, pl, st);
    }
}
template <typename T> cudaError_t launch(const AttendArgs &p, const Plan &pl, bool accumulate, cudaStream_t st) {
    if (!accumulate) return launch_dim<T, false>(p, pl, st);
    const cudaError_t e = launch_dim<T, true>(p, pl, st);
    if (e != cudaSuccess) return e;
    const int padded = pl.row_blocks * 8 * pl.nt;
    accumulate_kernel<2><<<pl.sms * 8, AT_THREADS, 0, st>>>(p, padded);
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

}  // namespace
}  // namespace abra

ABRA_ERROR_WORD_ACCESSOR(paged_attention_error_word)

extern "C" int64_t abra_paged_attention_workspace(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q,
                                                  int32_t flags) {
    int rc = abra::check(kv, n_heads, n_q, flags);
    if (rc) return rc;
    abra::Plan pl;
    rc = abra::make_plan(kv, n_heads, n_q, flags & ABRA_PAGED_ACCUMULATE, pl);
    return rc ? rc : pl.bytes;
}

extern "C" int abra_paged_attention(const abra_paged_kv *kv, const void *q, int64_t ldq, int32_t n_heads,
                                    int32_t n_q, float scale, void *out, int32_t out_type, int64_t ldo,
                                    float *lse, int32_t flags, void *workspace, int64_t workspace_bytes,
                                    void *stream) {
    using namespace abra;
    int rc = check(kv, n_heads, n_q, flags);
    if (rc) return rc;
    if (out_type != kv->type && out_type != ABRA_GGML_F32)
        return paged_fail(ABRA_E_UNSUPPORTED, "out must be of the cache's type or F32 (got %d)", out_type);
    if (!q || !out || !workspace) return paged_fail(ABRA_E_INVALID, "null q, out or workspace");
    if (ldq < static_cast<int64_t>(n_heads) * kv->head_dim || ldo < static_cast<int64_t>(n_heads) * kv->head_dim)
        return paged_fail(ABRA_E_INVALID, "a row stride is smaller than its heads");
    if (ldq % 8 || ldo % 8 || !paged_aligned(q, 16) || !paged_aligned(out, 16) || !paged_aligned(lse, 4))
        return paged_fail(ABRA_E_INVALID, "q and out rows must start on 16 bytes and their strides be multiples of 8 elements");
    if (!paged_aligned(workspace, 256)) return paged_fail(ABRA_E_INVALID, "the workspace must be 256-byte aligned");
    if (workspace_bytes < 256) return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes", (long long)workspace_bytes);
    if (kv->n_seqs == 0) return ABRA_OK;
    const bool accumulate = flags & ABRA_PAGED_ACCUMULATE;
    Plan pl;
    rc = make_plan(kv, n_heads, n_q, accumulate, pl);
    if (rc) return rc;
    if (workspace_bytes < pl.bytes)
        return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)pl.bytes);
    char *ws = static_cast<char *>(workspace);
    const int group = n_heads / kv->n_kv_heads;
    AttendArgs p{paged_view(kv),
                 q,
                 out,
                 lse,
                 ldq,
                 ldo,
                 scale * 1.4426950408889634f,
                 n_heads,
                 n_q,
                 group,
                 group * n_q,
                 pl.row_blocks,
                 out_type == ABRA_GGML_F32,
                 reinterpret_cast<unsigned *>(ws + pl.arrived),
                 reinterpret_cast<float *>(ws + pl.part_o),
                 reinterpret_cast<float2 *>(ws + pl.part_ml),
                 accumulate ? reinterpret_cast<float *>(ws + pl.row_lse) : nullptr,
                 reinterpret_cast<float *>(ws + pl.scores)};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return paged_cuda(kv->type == ABRA_GGML_F16 ? launch<__half>(p, pl, accumulate, st)
                                                : launch<__nv_bfloat16>(p, pl, accumulate, st),
                      "paged attention launch");
}
