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
// (sequence, kv head, block of rows) triples form one line, cut into equal
// pieces of one CTA each, which cross from triple to triple.  There are several
// pieces to a resident CTA where there is enough work, because CTAs with the
// same bytes to read finish at very different times (43 to 93 us of one
// 131,071-slot sequence in 444 equal pieces).  A second kernel joins the rows
// that were split and adds the weights.
//
// Layout: both products run on the tensor cores with the slots (16 a warp) as
// the tall side and the rows (8 a tile) as the narrow one, S^T = K Q^T and O^T
// = V^T P^T, so that a group of four heads wastes half a tile and not three
// quarters.  Each warp has a ring of tiles of its own in shared memory, filled
// by asynchronous 16-byte copies (zeros past the end) that run ahead across the
// ends of the rows; no warp waits for another before a row ends.
//
// Measured (B200, 1965 MHz, groups of four heads of 128): 64 sequences of up to
// 16,384 slots, 1.06 GB, 179 us = 5.9 TB/s, 0.91 of the measured HBM copy; one
// of 131,071, 0.54 GB, 94 us = 5.7 TB/s; 32 of up to 4,096, 65 MB, 21 us; one of
// 600, 8.9 us, of which 3 are the join's.  DRAM reads are the cache's bytes
// (537.0 of 536.9 MB); issue slots 40 % used, tensor pipe 12 %.
#include <algorithm>

#include "paged_attention.cuh"

namespace abra {
namespace {

constexpr int AT_WARPS = 4, AT_THREADS = AT_WARPS * 32;
constexpr int TILE = 16;               // slots of a warp's tile
constexpr int STEP = TILE * AT_WARPS;  // slots of a CTA's step

// ------------------------------------------------------------------ PTX ---
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
// Four 8x8 matrices of 16-bit values, lane l naming row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldm_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
// Transpose of an 8x8 matrix of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// --------------------------------------------------------------- kernel ---
// Rows of a block.  More rows a kv head go to paged_attention_wide.cu, which reads
// the slots once for 16 to 64 of them: 16 rows over 131,072 slots 99 us there, 153
// here in two blocks; 32 sequences of up to 8,192 33 and 40.  With many short
// sequences its rows' ends cost more than that gains (64 of up to 512 slots 26.9
// there, 25.1 here; 128 of up to 1,000 55.6 and 49.2), but lengths are on the
// device when the kernel is chosen.  Up to eight rows are one block here, and
// faster (four rows, 32 sequences of up to 4,096 slots: 18.0 us here, 24.7 there).
constexpr int ROWS = 8;
constexpr int CTAS = 3;   // on a multiprocessor, with rings of two tiles (two CTAs with rings of three: 188 against 179 us for
                          // 64 sequences of up to 16,384 slots, 24 against 21 for 32 of up to 4,096)
template <int D> struct Shape {
    static constexpr int KS = D / 16;           // k-steps of the scores, and 16-element tiles of the output
    static constexpr int CHUNKS = D / 8;        // 16-byte chunks of a row
    static constexpr int COPIES = CHUNKS / 2;   // of a lane for a tile of 16 rows
    // A row's chunk c lies at c ^ (row % 8), where the chunks are 8 or 16; rows
    // of 12 are padded by one instead.  Either way the eight rows of an ldmatrix
    // lie in distinct banks.
    static constexpr bool SWIZZLE = D != 96;
    static constexpr int ROW = SWIZZLE ? 2 * D : 2 * D + 16;  // bytes of a row in the ring
    static constexpr int TILE_BYTES = TILE * ROW;             // K or V of one tile
    static constexpr int STAGE = AT_WARPS * 2 * TILE_BYTES;   // the CTA's K and V tiles
    static constexpr int PITCH = D + 4;                       // floats of a row in a join buffer
    static constexpr int JOIN_BYTES = 2 * ROWS * PITCH * 4 + 2 * AT_WARPS * ROWS * 4 + ROWS * D / 4;
    // the ring: as many tiles as leave room for the CTAs (1 KB each is the system's)
    static constexpr int DEPTH = (233472 / CTAS - 1024 - 256 - JOIN_BYTES) / STAGE;
    static constexpr int SMEM = DEPTH * STAGE + JOIN_BYTES;
    static_assert(DEPTH >= 2, "the ring needs two tiles");
    static __device__ __forceinline__ int at(int row, int chunk) { return row * ROW + ((SWIZZLE ? chunk ^ (row & 7) : chunk) << 4); }
    // `bytes` (a multiple of 32) along a row from the chunk at `a`, an even chunk or the one behind it
    static __device__ __forceinline__ uint32_t along(uint32_t a, int bytes) { return SWIZZLE ? a ^ bytes : a + bytes; }
};

template <typename T, int D, bool SCORES>
__global__ void __launch_bounds__(AT_THREADS, CTAS) attend_kernel(const __grid_constant__ AttendArgs p) {
    using S = Shape<D>;
    extern __shared__ __align__(256) unsigned char smem[];  // the ring: [warp][stage][K, V][row]
    float *s_o = reinterpret_cast<float *>(smem + S::DEPTH * S::STAGE);  // [2][ROWS][PITCH]
    float *s_m = s_o + 2 * ROWS * S::PITCH, *s_l = s_m + AT_WARPS * ROWS;  // [warp][ROWS]
    uint32_t *s_saw = reinterpret_cast<uint32_t *>(s_l + AT_WARPS * ROWS);  // [ROWS][D] codes of two bits
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;

    pdl_wait();
    pdl_launch_dependents();  // the join may take its place; it waits for the whole grid
    Walk<STEP> w;
    Line line(0, 0);
    if (!find_start<AT_THREADS>(p.kv, p.row_blocks, blockIdx.x, gridDim.x, p.resident, line, w)) return;
    const int begin = w.pos;

    // ---- the fetching side: this warp's tiles, segment after segment ----
    // Copy i of a lane moves 16-byte chunk (32 i + lane) % CHUNKS of row (32 i +
    // lane) / CHUNKS; the first half of the copies are rows 0-7, the second
    // rows 8-15.  Where eight divides the page size each half lies in one page.
    const uint32_t ring = smem_u32(smem) + warp * (S::DEPTH * 2 * S::TILE_BYTES);
    const bool by8 = p.kv.a.page_size % 8 == 0;
    Walk<STEP> f = w;
    int f_base = f.s.tile0 * STEP + warp * TILE, f_valid = 0;
    // (a table entry for every tile where eight does not divide the page size: 32
    // sequences of up to 4,096 slots 18.5 us with pages of 7, 18.1 with 16)
    int f_page = 0;    // of half l % 2 of the batch's tile l / 2, or (by8 false) of row l % 16 of this tile
    int f_tile = 16;   // this tile's place in its batch of 16; 16: the next batch is to be read
    uint32_t f_at = ring;
    bool f_more = true;
    int64_t f_v0 = 0, f_v1 = 0;  // V offsets of the halves' first rows, or (by8 false) f_v0 of row lane % 16
    auto page_of = [&](int t) {
        return t < f.s.slot_end ? p.kv.a.table[static_cast<int64_t>(f.s.seq) * p.kv.a.table_stride + p.kv.page.div(t)] : 0;
    };
    auto fetch_settle = [&]() {  // on to the next tile that exists, and its pages
        while (f_base >= f.s.slot_end) {
            f_more = f.next(p.kv);
            if (!f_more) return;
            f_base = f.s.tile0 * STEP + warp * TILE;
            f_tile = 16;
        }
        if (!by8) {
            f_page = page_of(f_base + (lane & 15));
        } else if (f_tile == 16) {
            f_page = page_of(f_base + (lane >> 1) * STEP + 8 * (lane & 1));
            f_tile = 0;
        }
    };
    auto in_pool = [&](int &page) {
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.kv.a.n_pages)) {
            report_error(ERR_BAD_INDEX);
            page = 0;
        }
    };
    auto copy_tile = [&](const T *pool, int64_t off0, int64_t off1, int64_t stride, uint32_t to) {
        const T *src0 = pool + off0, *src1 = pool + off1;
#pragma unroll
        for (int i = 0; i < S::COPIES; ++i) {
            const int x = 32 * i + lane, row = x / S::CHUNKS, chunk = x - row * S::CHUNKS;
            const T *src;
            if (by8)
                src = (2 * i < S::COPIES ? src0 : src1) + (row & 7) * stride;
            else
                src = pool + __shfl_sync(0xffffffffu, off0, row);
            copy_async(to + S::at(row, chunk), src + chunk * 8, row < f_valid ? 16 : 0);
        }
    };
    auto fetch_k = [&]() {
        f_valid = 0;
        if (f_more) {
            f_valid = f.s.slot_end - f_base;
            const int t0 = by8 ? f_base : f_base + (lane & 15), off0 = t0 - p.kv.page.div(t0) * p.kv.a.page_size;
            int page0 = by8 ? __shfl_sync(0xffffffffu, f_page, 2 * f_tile) : f_page;
            in_pool(page0);
            const int64_t k0 = paged_k_at(p.kv, page0, f.s.head, off0);
            f_v0 = paged_v_at(p.kv, page0, f.s.head, off0);
            int64_t k1 = 0;
            if (by8) {
                const int off1 = f_base + 8 - p.kv.page.div(f_base + 8) * p.kv.a.page_size;
                int page1 = __shfl_sync(0xffffffffu, f_page, 2 * f_tile + 1);
                in_pool(page1);
                k1 = paged_k_at(p.kv, page1, f.s.head, off1);
                f_v1 = paged_v_at(p.kv, page1, f.s.head, off1);
                ++f_tile;
            }
            copy_tile(static_cast<const T *>(p.kv.a.k), k0, k1, p.kv.a.k_slot_stride, f_at);
        }
        copy_commit();
    };
    auto fetch_v = [&]() {
        if (f_valid > 0) {
            copy_tile(static_cast<const T *>(p.kv.a.v), f_v0, f_v1, p.kv.a.v_slot_stride, f_at + S::TILE_BYTES);
            f_base += STEP;
            fetch_settle();
        }
        copy_commit();
        f_at += 2 * S::TILE_BYTES;
        if (f_at == ring + S::DEPTH * 2 * S::TILE_BYTES) f_at = ring;
    };
    fetch_settle();
#pragma unroll 1
    for (int i = 0; i < S::DEPTH; ++i) {
        fetch_k();
        fetch_v();
    }
    // this lane's row of an ldmatrix: K's matrices are (slots 0-7, 8-15) x
    // (elements 0-7, 8-15) in the order of an A fragment; V's are transposed, so
    // slots and elements change places
    const uint32_t k_lane = S::at(lane & 15, lane >> 4);
    const uint32_t v_lane = S::TILE_BYTES + S::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
    uint32_t at = ring;

    do {
        const Segment &sg = w.s;
        const int head = sg.head;

        // Q fragments: row g, elements 16 ks + 2 c and + 8; rows past the end are zeros
        uint2 qf[S::KS];
        {
            const int j = min(g, p.rows - 1) / p.group, h = head * p.group + g - j * p.group;
            const T *q = static_cast<const T *>(p.q) + (static_cast<int64_t>(sg.seq) * p.n_q + j) * p.ldq + static_cast<int64_t>(h) * D + 2 * c;
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks)
                qf[ks] = g < p.rows ? make_uint2(*reinterpret_cast<const unsigned *>(q + 16 * ks),
                                                 *reinterpret_cast<const unsigned *>(q + 16 * ks + 8))
                                    : make_uint2(0, 0);
        }
        // slots below are seen by every row; row 2 c + e sees `seen` of them
        const int all_see = sg.len - p.n_q + 1;
        auto seen = [&](int e) { return all_see + min((2 * c + e) / p.group, p.n_q - 1); };

        // running maximum m of each row (and 0 in its place while it is -infinity), sum, result
        float o[S::KS][4], m[2], sub[2], l[2];
#pragma unroll
        for (int mt = 0; mt < S::KS; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.0f;
        m[0] = m[1] = -INFINITY;
        sub[0] = sub[1] = l[0] = l[1] = 0.0f;
        bool odd = false;  // an infinity or NaN was taken out of a tile
        const int64_t seq_scores = SCORES ? score_at(p, sg.seq, head, 0, -1) : 0;

        for (int base = sg.tile0 * STEP + warp * TILE; base < sg.slot_end; base += STEP) {
            // scores: slots g, g + 8 of the tile by rows 2c, 2c + 1; two sums, for
            // two chains of half the length
            float sc[4], part[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) part[x][0] = part[x][1] = part[x][2] = part[x][3] = 0.0f;
            copy_wait<2 * S::DEPTH - 1>();
            __syncwarp();
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks) {
                uint32_t a[4];
                ldm(a, S::along(at + k_lane, ks * 32));
                mma_16x8x16<T>(part[ks & 1], a[0], a[1], a[2], a[3], qf[ks].x, qf[ks].y);
            }
            __syncwarp();
            fetch_k();  // into the tile just read
            // log2 units, the mask, and the rows' maxima
            const bool edge = base + TILE > all_see;
            bool raise = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[e] = (part[0][e] + part[1][e]) * p.scale_log2;
                if (edge && base + g + 8 * (e >> 1) >= seen(e & 1)) sc[e] = -INFINITY;
                raise |= sc[e] - m[e & 1] > Weigh<T>::RAISE;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(sc[e], sc[e + 2]);
#pragma unroll
                    for (int x = 4; x <= 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    top = fmaxf(top, m[e]);
                    const float k = scaled(m[e], top);
                    m[e] = top;
                    sub[e] = top == -INFINITY ? 0.0f : top;
                    l[e] *= k;
#pragma unroll
                    for (int mt = 0; mt < S::KS; ++mt) o[mt][e] *= k, o[mt][e + 2] *= k;
                }
            }
            if (SCORES) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int t = base + g + 8 * x, e = p.kv.page.div(t);
                    const int page = t < sg.slot_end ? paged_page(p.kv, sg.seq, e) : -1;
                    if (page >= 0) {  // a page outside the pool has no place for them
                        float *to = p.scores + (seq_scores < 0 ? paged_meta_at(p.kv, page, head, t - e * p.kv.a.page_size) : seq_scores + t) * ROWS;
                        *reinterpret_cast<float2 *>(to + 2 * c) = make_float2(sc[2 * x], sc[2 * x + 1]);
                    }
                }
            }
            // weights, as the sum of two 16-bit values: the tensor cores take
            // 16-bit operands, and one rounding would cost as much precision
            // as the result's own
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[e] = weight_of<T>(sc[e], sub[e & 1]);
                l[e & 1] += sc[e];
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t h = pack2<T>(sc[2 * x], sc[2 * x + 1]);
                const float2 r = unpack2<T>(h);
                hi[x] = trans8x8(h);
                lo[x] = trans8x8(pack2<T>(sc[2 * x] - r.x, sc[2 * x + 1] - r.y));
            }
            copy_wait<2 * S::DEPTH - 1>();
            __syncwarp();
            if (edge && p.n_q > 1) {  // not every row sees them all: look_through
#pragma unroll 1
                for (int i = 0; i < S::COPIES; ++i) {
                    const int x = 32 * i + lane, row = x / S::CHUNKS, chunk = x - row * S::CHUNKS;
                    uint4 *v = reinterpret_cast<uint4 *>(smem + (at - smem_u32(smem)) + S::TILE_BYTES + S::at(row, chunk));
                    bool any = false;
                    const uint4 y = make_uint4(finite_part<T>(v->x, any), finite_part<T>(v->y, any), finite_part<T>(v->z, any),
                                               finite_part<T>(v->w, any));
                    if (any) *v = y, odd = true;
                }
                __syncwarp();
            }
#pragma unroll
            for (int mt = 0; mt < S::KS; ++mt) {
                uint32_t a[4];
                ldm_trans(a, S::along(at + v_lane, mt * 32));
                mma_16x8x16<T>(o[mt], a[0], a[1], a[2], a[3], hi[0], hi[1]);
                mma_16x8x16<T>(o[mt], a[0], a[1], a[2], a[3], lo[0], lo[1]);
            }
            __syncwarp();
            fetch_v();
            at += 2 * S::TILE_BYTES;
            if (at == ring + S::DEPTH * 2 * S::TILE_BYTES) at = ring;
        }

        // ---- join the warps: maxima, then the scaled sums, two warps after two ----
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
            if (g == 0) s_m[warp * ROWS + 2 * c + e] = m[e], s_l[warp * ROWS + 2 * c + e] = l[e];
        }
        // a NaN that the row's weights do not explain comes from the values
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int mt = 0; mt < S::KS; ++mt) sum[0] += o[mt][e], sum[1] += o[mt][e + 2];
            odd |= isnan(sum[0] + sum[1]) && !isnan(l[e]);
        }
        odd = __syncthreads_or(odd);
        auto top_of = [&](int r) {
            float top = s_m[r];
#pragma unroll
            for (int x = 1; x < AT_WARPS; ++x) top = fmaxf(top, s_m[x * ROWS + r]);
            return top;
        };
#pragma unroll 1
        for (int turn = 0; turn < AT_WARPS / 2; ++turn) {
            if (warp >> 1 == turn) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 2 * c + e;
                    const float k = scaled(m[e], top_of(r));
                    float *dst = s_o + ((warp & 1) * ROWS + r) * S::PITCH + g;
#pragma unroll
                    for (int mt = 0; mt < S::KS; ++mt)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float x = o[mt][e + 2 * y] * k;
                            dst[16 * mt + 8 * y] = turn ? dst[16 * mt + 8 * y] + x : x;
                        }
                }
            }
            __syncthreads();
        }
        if (odd) {
            for (int i = tid; i < ROWS * D / 16; i += AT_THREADS) s_saw[i] = 0;
            __syncthreads();
            look_through<T, D, AT_THREADS>(p, sg.seq, head, sg.tile0 * STEP, sg.slot_end, all_see, 0, p.rows, tid, s_saw);
            __syncthreads();
        }
        const bool whole = sg.tile0 == 0 && sg.tile1 == sg.n;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (w.pos == begin ? 0 : 1);
        for (int i = tid; i < ROWS * (D / 4); i += AT_THREADS) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            if (r >= p.rows) break;
            const float top = top_of(r);
            float total = 0.0f;
#pragma unroll
            for (int x = 0; x < AT_WARPS; ++x) total += s_l[x * ROWS + r] * scaled(s_m[x * ROWS + r], top);
            float4 sum = *reinterpret_cast<const float4 *>(s_o + r * S::PITCH + d);
            const float4 y = *reinterpret_cast<const float4 *>(s_o + (ROWS + r) * S::PITCH + d);
            sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
            if (odd) {
                const int at = r * D + d;
                sum = make_float4(with_saw(sum.x, s_saw, at), with_saw(sum.y, s_saw, at + 1), with_saw(sum.z, s_saw, at + 2),
                                  with_saw(sum.w, s_saw, at + 3));
            }
            if (whole) {
                finish_row<T>(p, sg.seq, head, r, d, D, sum, top, total);
            } else {
                *reinterpret_cast<float4 *>(p.part_o + (slot * ROWS + r) * D + d) = sum;
                if (d == 0) p.part_ml[slot * ROWS + r] = make_float2(top, total);
            }
        }
        if (sg.tile0 == 0 && tid == 0)
            p.split[static_cast<int64_t>(sg.seq) * w.units + sg.unit] =
                make_int2(static_cast<int>(slot), whole ? static_cast<int>(blockIdx.x) : line.piece(sg.row_begin + ROW_COST + sg.n - 1));
        __syncthreads();  // the join buffers are free again
    } while (w.next(p.kv));
}

// Parts of a row: the first at place `first` (a piece has two), then one in the
// first place of each piece up to `last`.
struct Parts {
    int first, last;
    __device__ __forceinline__ Parts(int2 x) : first(x.x), last(x.y) {}
    __device__ __forceinline__ int count() const { return last - (first >> 1) + 1; }
    __device__ __forceinline__ int64_t place(int i) const { return i ? 2 * (static_cast<int64_t>(first >> 1) + i) : first; }
};

constexpr int JOIN_WARPS = 8, JOIN_THREADS = JOIN_WARPS * 32;
constexpr int ACC_ROWS = 64;  // rows whose lse is held at a time
// CTAs that accumulate, on a multiprocessor; four of them fit, and those that
// join come behind them (the other way round, with two lanes a slot and three
// CTAs: 36 against 32 us for 16 sequences of up to 8,192 slots, 64 heads).
constexpr int ACC_CTAS = 4;

struct JoinArgs {
    AttendArgs a;
    int block;         // rows of a block
    int warps;         // of an output row: 1, 2, 4 or 8
    int row_ctas;      // CTAs for the rows of one kv head of a sequence
    int joins;         // CTAs that join; the others accumulate
};

// CTA `cta`: JOIN_WARPS / warps output rows.  The parts of a row are dealt to
// its warps, which meet in shared memory in a fixed order.
template <typename T, int D> __device__ __forceinline__ void join_rows(const JoinArgs &ja, int cta) {
    const AttendArgs &p = ja.a;
    __shared__ float s_top[JOIN_WARPS], s_total[JOIN_WARPS];
    __shared__ __align__(16) float s_sum[JOIN_WARPS][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = cta / ja.row_ctas, head = group % p.kv.a.n_kv_heads, seq = group / p.kv.a.n_kv_heads;
    const int row = warp / ja.warps, part = warp - row * ja.warps;
    const int r = (cta - group * ja.row_ctas) * (JOIN_WARPS / ja.warps) + row;
    const bool in = r < p.rows;
    const int len = paged_len(p.kv, seq), block = in ? r / ja.block : 0, rr = r - block * ja.block;
    // (of an empty sequence nobody wrote this, and nobody looks at it)
    const Parts parts(__ldcg(p.split + (static_cast<int64_t>(seq) * p.kv.a.n_kv_heads + head) * p.row_blocks + block));
    const int n = in && len > 0 ? parts.count() : 1;  // one part: the row is done
    float top = -INFINITY, total = 0.0f;
    float4 sum = make_float4(0, 0, 0, 0);
    // this warp's parts: part, part + warps, ..., 32 of them at a time
    for (int base = part; n > 1 && base < n; base += 32 * ja.warps) {
        const int mine = base + lane * ja.warps;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (mine < n) ml = __ldcg(p.part_ml + parts.place(mine) * ja.block + rr);
        const int left = min(32, (n - base + ja.warps - 1) / ja.warps);
        // all parts but the first lie evenly; eight loads in flight a lane
        const int64_t even = (2 * (static_cast<int64_t>(parts.first >> 1) + base) * ja.block + rr) * D;
        const int64_t odd = base == 0 ? (static_cast<int64_t>(parts.first & 1)) * ja.block * D : 0;
        const float *src = p.part_o + even + 4 * min(lane, D / 4 - 1);
        float k = 0.0f;
        for (int i0 = 0; i0 < left; i0 += 8) {
            float4 y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = make_float4(0, 0, 0, 0);
                if (i0 + i < left)
                    y[i] = __ldcg(reinterpret_cast<const float4 *>(src + (i0 + i == 0 ? odd : 0) +
                                                                   static_cast<int64_t>(i0 + i) * (2 * D) * ja.warps * ja.block));
            }
            if (i0 == 0) {
                float t = ml.x;
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                t = fmaxf(t, top);
                const float keep = scaled(top, t);
                k = scaled(ml.x, t);
                top = t;
                total = total * keep + ml.y * k;  // lane by lane, added up below
                sum.x *= keep, sum.y *= keep, sum.z *= keep, sum.w *= keep;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float ki = __shfl_sync(0xffffffffu, k, i0 + i);  // meets zeros beyond the last part
                sum.x += ki * y[i].x, sum.y += ki * y[i].y, sum.z += ki * y[i].z, sum.w += ki * y[i].w;
            }
        }
    }
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    if (ja.warps > 1) {
        if (lane == 0) s_top[warp] = top, s_total[warp] = total;
        if (lane < D / 4) *reinterpret_cast<float4 *>(&s_sum[warp][4 * lane]) = sum;
        __syncthreads();
        if (part) return;
        top = s_top[warp];
        const int used = min(n, ja.warps);
        for (int x = 1; x < used; ++x) top = fmaxf(top, s_top[warp + x]);
        total = 0.0f;
        sum = make_float4(0, 0, 0, 0);
        for (int x = 0; x < used; ++x) {
            const float k = scaled(s_top[warp + x], top);
            const float4 y = *reinterpret_cast<const float4 *>(&s_sum[warp + x][4 * min(lane, D / 4 - 1)]);
            total += s_total[warp + x] * k;
            sum.x += k * y.x, sum.y += k * y.y, sum.z += k * y.z, sum.w += k * y.w;
        }
    }
    if (in && (n > 1 || len == 0) && lane < D / 4) finish_row<T>(p, seq, head, r, 4 * lane, D, sum, top, total);
}

// acc += the slots' weights, exp2(score - lse) summed over the rows, on pieces
// of the same kind of line; a lane takes eight rows of a slot, as many lanes a
// slot as a block has eights.  A row's lse comes from its parts, so this needs
// the first kernel only.
template <typename T> __device__ __forceinline__ void accumulate(const JoinArgs &ja, int cta, int ctas) {
    const AttendArgs &p = ja.a;
    __shared__ __align__(16) float s_lse[ACC_ROWS];
    const int tid = threadIdx.x, heads = p.kv.a.n_kv_heads, lanes = ja.block / 8, slots = JOIN_THREADS / lanes;
    const int mine = 8 * (tid % lanes), padded = p.row_blocks * ja.block;
    Walk<STEP> w;
    Line line(0, 0);
    if (!find_start<JOIN_THREADS>(p.kv, 1, cta, ctas, ctas, line, w)) return;
    // rows that see nothing, and what lies behind the last row, have an lse of +infinity and no weight;
    // nor has a slot that a row does not see, whose own lse may be NaN
    auto weight = [](float x, float lse) { return lse == INFINITY || x == -INFINITY ? 0.0f : exp2_fast(x - lse); };
    do {
        const Segment &sg = w.s;
        const int first = sg.tile0 * STEP + tid / lanes;  // this thread's slot, and every `slots` after it
        const int64_t seq_scores = score_at(p, sg.seq, sg.head, 0, -1);  // of slot 0, or -1: they lie as the pages do
        auto page_of = [&](int t) { return t < sg.slot_end ? paged_page(p.kv, sg.seq, p.kv.page.div(t)) : -1; };
        for (int r0 = 0; r0 < p.rows; r0 += ACC_ROWS) {
            const int nr = min(ACC_ROWS, p.rows - r0);
            int page = page_of(first);  // runs beside the rows' lse
            __syncthreads();
            if (tid < ACC_ROWS && tid >= nr) s_lse[tid] = INFINITY;
            for (int i = tid >> 5; i < nr; i += JOIN_WARPS) {  // a warp a row
                const int r = r0 + i, block = r / ja.block;
                const int64_t triple = (static_cast<int64_t>(sg.seq) * heads + sg.head);
                const Parts parts(__ldcg(p.split + triple * p.row_blocks + block));
                const int n = parts.count(), lane = tid & 31;
                float lse;
                if (n == 1) {
                    lse = __ldcg(p.row_lse + triple * p.rows + r);
                } else {
                    float top = -INFINITY, total = 0.0f;
                    for (int x = lane; x < n; x += 32) {
                        const float2 ml = __ldcg(p.part_ml + parts.place(x) * ja.block + r - block * ja.block);
                        const float t = fmaxf(top, ml.x);
                        total = total * scaled(top, t) + ml.y * scaled(ml.x, t);
                        top = t;
                    }
#pragma unroll
                    for (int x = 16; x >= 1; x >>= 1) {
                        const float ot = __shfl_xor_sync(0xffffffffu, top, x), on = __shfl_xor_sync(0xffffffffu, total, x);
                        const float t = fmaxf(top, ot);
                        total = total * scaled(top, t) + on * scaled(ot, t);
                        top = t;
                    }
                    lse = row_lse2<T>(top, total);
                }
                if (lane == 0) s_lse[i] = lse == -INFINITY ? INFINITY : lse;
            }
            __syncthreads();
            for (int t = first; t - tid / lanes < sg.slot_end; t += slots) {
                const int64_t meta = page < 0 ? -1 : paged_meta_at(p.kv, page, sg.head, t - p.kv.page.div(t) * p.kv.a.page_size);
                const float acc = meta >= 0 && mine == 0 ? p.kv.a.acc[meta] : 0.0f;
                float4 x[2];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    x[y] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (meta >= 0 && mine + 4 * y < nr)
                        x[y] = __ldcg(reinterpret_cast<const float4 *>(p.scores + (seq_scores < 0 ? meta : seq_scores + t) * padded + r0 + mine + 4 * y));
                }
                page = page_of(t + slots);
                float sum = 0.0f;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float4 lse = *reinterpret_cast<const float4 *>(s_lse + mine + 4 * y);
                    sum += weight(x[y].x, lse.x) + weight(x[y].y, lse.y) + weight(x[y].z, lse.z) + weight(x[y].w, lse.w);
                }
                for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (meta >= 0 && mine == 0) p.kv.a.acc[meta] = acc + sum;
            }
        }
    } while (w.next(p.kv));
}

// The second kernel: it writes the rows of empty sequences (zeros), joins the
// rows that were split, and adds the slots' weights, side by side.
template <typename T, int D, bool SCORES> __global__ void __launch_bounds__(JOIN_THREADS, SCORES ? 4 : 3) join_kernel(const __grid_constant__ JoinArgs ja) {
    pdl_wait();
    pdl_launch_dependents();
    const int cta = blockIdx.x;
    const int adding = SCORES ? gridDim.x - ja.joins : 0;
    if (SCORES && cta < adding) accumulate<T>(ja, cta, adding);
    else join_rows<T, D>(ja, cta - adding);
}

// ------------------------------------------------------------------ host ---
struct Plan {
    int wide, block, row_blocks, resident, pieces, sms;  // block: rows of a block
    int score_slots;                                         // of a sequence's scores, 0: they lie as the pools do
    int64_t part_o, part_ml, split, row_lse, scores, bytes;  // workspace offsets
};

int make_plan(const abra_paged_kv *kv, int32_t n_heads, int32_t n_q, bool accumulate, Plan &pl) {
    pl.sms = device_sm_count();
    const int rows = n_heads / kv->n_kv_heads * n_q;
    pl.wide = rows > ROWS;
    pl.block = !pl.wide ? ROWS : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    pl.row_blocks = (rows + pl.block - 1) / pl.block;
    const int64_t triples = static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads * pl.row_blocks;
    const int step = pl.wide ? WIDE_STEP : STEP;
    const int64_t steps = (static_cast<int64_t>(kv->max_pages) * kv->page_size + step - 1) / step + ROW_COST;
    if (steps * triples > 0x7fffffff || static_cast<int64_t>(kv->n_seqs) * n_heads * n_q > 0x3fffffff)
        return paged_fail(ABRA_E_UNSUPPORTED, "over 2^31 steps of %d slots in the tables, or over 2^30 output rows", step);
    pl.resident = pl.sms * (pl.wide ? 1 : CTAS);
    pl.pieces = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(pl.resident) * (pl.wide ? 1 : WAVES), steps * triples));
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    int64_t at = 0;
    pl.part_o = at, at = up(at + static_cast<int64_t>(pl.pieces) * 2 * pl.block * kv->head_dim * 4);
    pl.part_ml = at, at = up(at + static_cast<int64_t>(pl.pieces) * 2 * pl.block * 8);
    pl.split = at, at = up(at + triples * 8);
    pl.row_lse = pl.scores = at;
    const int64_t tables = static_cast<int64_t>(kv->n_seqs) * kv->max_pages;
    pl.score_slots = tables < kv->n_pages ? kv->max_pages * kv->page_size : 0;
    if (accumulate) {
        at = up(at + static_cast<int64_t>(kv->n_seqs) * kv->n_kv_heads * rows * 4);
        pl.scores = at;
        at = up(at + std::min<int64_t>(tables, kv->n_pages) * kv->n_kv_heads * kv->page_size * pl.row_blocks * pl.block * 4);
    }
    pl.bytes = at;
    return ABRA_OK;
}

template <typename T, int D, bool SCORES> cudaError_t launch_narrow(const AttendArgs &p, const Plan &pl, cudaStream_t st) {
    constexpr int smem = Shape<D>::SMEM;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = paged_smem(reinterpret_cast<const void *>(attend_kernel<T, D, SCORES>), smem, done);
    if (e != cudaSuccess) return e;
    return paged_launch(attend_kernel<T, D, SCORES>, dim3(pl.pieces), AT_THREADS, smem, st, p);
}
template <typename T, int D> cudaError_t launch_all(const AttendArgs &p, const Plan &pl, bool accumulate, cudaStream_t st) {
    cudaError_t e = pl.wide ? launch_attend_wide(p, pl.block, pl.pieces, accumulate, st)
                    : accumulate ? launch_narrow<T, D, true>(p, pl, st)
                                 : launch_narrow<T, D, false>(p, pl, st);
    if (e != cudaSuccess) return e;
    // as many warps a row as keep four CTAs' worth on every multiprocessor
    const int64_t groups = static_cast<int64_t>(p.kv.a.n_seqs) * p.kv.a.n_kv_heads;
    int warps = JOIN_WARPS;
    while (warps > 1 && groups * p.rows * warps > pl.sms * 4 * JOIN_WARPS) warps /= 2;
    const int per = JOIN_WARPS / warps, row_ctas = (p.rows + per - 1) / per;
    const JoinArgs ja{p, pl.block, warps, row_ctas, static_cast<int>(groups * row_ctas)};
    return accumulate ? paged_launch(join_kernel<T, D, true>, dim3(ja.joins + pl.sms * ACC_CTAS), JOIN_THREADS, 0, st, ja)
                      : paged_launch(join_kernel<T, D, false>, dim3(ja.joins), JOIN_THREADS, 0, st, ja);
}
template <typename T> cudaError_t launch(const AttendArgs &p, const Plan &pl, bool accumulate, cudaStream_t st) {
    switch (p.kv.a.head_dim) {
        case 64: return launch_all<T, 64>(p, pl, accumulate, st);
        case 96: return launch_all<T, 96>(p, pl, accumulate, st);
        default: return launch_all<T, 128>(p, pl, accumulate, st);
    }
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
    if (kv->n_seqs == 0) return ABRA_OK;
    if (!q || !out || !workspace) return paged_fail(ABRA_E_INVALID, "null q, out or workspace");
    if (ldq < static_cast<int64_t>(n_heads) * kv->head_dim || ldo < static_cast<int64_t>(n_heads) * kv->head_dim)
        return paged_fail(ABRA_E_INVALID, "a row stride is smaller than its heads");
    if (ldq % 8 || ldo % 8 || !paged_aligned(q, 16) || !paged_aligned(out, 16) || !paged_aligned(lse, 4))
        return paged_fail(ABRA_E_INVALID, "q and out rows must start on 16 bytes and their strides be multiples of 8 elements");
    if (!paged_aligned(workspace, 256)) return paged_fail(ABRA_E_INVALID, "the workspace must be 256-byte aligned");
    if (workspace_bytes < 256) return paged_fail(ABRA_E_INVALID, "workspace of %lld bytes", (long long)workspace_bytes);
    // rows are finished while others' queries are still to be read
    const int64_t width = static_cast<int64_t>(n_heads) * kv->head_dim, out_bytes = out_type == ABRA_GGML_F32 ? 4 : 2;
    if (paged_overlap({q, 2 * width, 2 * ldq}, {out, out_bytes * width, out_bytes * ldo}, static_cast<int64_t>(kv->n_seqs) * n_q))
        return paged_fail(ABRA_E_INVALID, "out must not share q's memory");
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
                 pl.resident,
                 reinterpret_cast<float *>(ws + pl.part_o),
                 reinterpret_cast<float2 *>(ws + pl.part_ml),
                 reinterpret_cast<int2 *>(ws + pl.split),
                 accumulate ? reinterpret_cast<float *>(ws + pl.row_lse) : nullptr,
                 reinterpret_cast<float *>(ws + pl.scores),
                 pl.score_slots};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return paged_cuda(kv->type == ABRA_GGML_F16 ? launch<__half>(p, pl, accumulate, st)
                                                : launch<__nv_bfloat16>(p, pl, accumulate, st),
                      "paged attention launch");
}
