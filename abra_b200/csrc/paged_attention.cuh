// paged_attention.cuh -- what the kernels of the paged attention share: their
// arguments, the line of steps that their CTAs divide, and the end of a row.
#pragma once

#include "paged_kv.cuh"

namespace abra {

constexpr int PIECE = 16;                 // steps of a piece, where there are enough to fill the GPU (131,071 slots: 93 us;
                                          // with 8, and so twice the parts to join, 99)
constexpr int WAVES = 4;                  // pieces for each CTA that the GPU holds, at most; the wide kernel's CTA fills its
                                          // multiprocessor, so that nothing runs beside a new one's start, and takes one
// A row's weights are 2^(s - m + SHIFT) of its running maximum m, and so are its
// sums until its log-sum-exp takes SHIFT off again.  m is raised only when a score
// passes it by RAISE, so that most tiles need no reduction; weights stay below
// 2^(RAISE + SHIFT), for which compare and weight both take the difference s - m
// first (m + RAISE or m - SHIFT would be rounded where m is large).  fp16 ends at
// 2^-24, so its weights go up to the top of its range: of a weight at most 2^-36 of
// the row's largest is lost, without SHIFT 2^-25, which beside a slot far above the
// others is all of them.  RAISE 2 and SHIFT 13 raise more often than they are worth
// (16 new tokens of four sequences of up to 8,192 slots 26.5 us, 25.6 with 4 and 11,
// 25.4 with 10 and 5).  bf16 has fp32's range, in values too: its weights are so
// small that 2^22 of the largest values do not add up to infinity before the row is
// divided by its sum, and large enough for products of values above 2^-90.
template <typename T> struct Weigh;
template <> struct Weigh<__half> {
    static constexpr float RAISE = 4.0f;
    static constexpr int SHIFT = 11;
};
template <> struct Weigh<__nv_bfloat16> {
    static constexpr float RAISE = 10.0f;
    static constexpr int SHIFT = -32;
};
constexpr float power_of_two(int n) { return n < 0 ? 1.0f / power_of_two(-n) : n == 0 ? 1.0f : 2.0f * power_of_two(n - 1); }
// What beginning and ending a row costs beside its steps, in steps (its
// queries, the join of its warps): with 1 the pieces full of short rows end
// last (21.7 against 20.8 us for 32 sequences of 1 to 4,096 slots), with 3
// the long rows do (21.8).
constexpr int ROW_COST = 2;

struct AttendArgs {
    PagedKv kv;
    const void *q;
    void *out;
    float *lse;
    int64_t ldq, ldo;
    float scale_log2;  // scale / ln 2: scores are kept in units of log2
    int n_heads, n_q, group, rows, row_blocks, out_f32;
    int resident;  // CTAs of the first kernel that the GPU holds at once
    // workspace
    float *part_o;      // [piece][2][rows of a block][D]
    float2 *part_ml;    // [piece][2][rows of a block] maximum (log2 units) and sum
    int2 *split;        // [seq][kv head][row block] the first part's place, the last part's piece
    float *row_lse;     // [seq][kv head][row] log2 of the sum of a row that lies in one piece
    float *scores;      // [page][kv head][offset][padded rows], log2 units; or [seq][kv head][slot][padded rows]
    int score_slots;    // slots of a sequence in the latter, 0: the former
};

// A slot's place among the scores: that of its page, or its own in the tables where
// these name fewer slots than the pools have.
__device__ __forceinline__ int64_t score_at(const AttendArgs &p, int seq, int head, int t, int64_t meta) {
    return p.score_slots ? (static_cast<int64_t>(seq) * p.kv.a.n_kv_heads + head) * p.score_slots + t : meta;
}

// ------------------------------------------------------------------ PTX ---
// 16 bytes into shared memory past L1; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A score's weight against `ref`, the row's maximum (0 while that is -infinity).
// (a product, not a sum with SHIFT: s - ref keeps its bits)
template <typename T> __device__ __forceinline__ float weight_of(float s, float ref) { return exp2_fast(s - ref) * power_of_two(Weigh<T>::SHIFT); }
// What a sum relative to the maximum m counts relative to `top`; never zero, so
// that a sum of infinity stays one.
__device__ __forceinline__ float scaled(float m, float top) { return m == top ? 1.0f : exp2_fast(fmaxf(m - top, -126.0f)); }
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
struct Line {
    int total;       // the triples' costs
    int pieces;      // each has at least one unit of cost
    int quot, rest;  // total / pieces and what is left
    __device__ __forceinline__ Line(int total, int pieces) : total(total), pieces(pieces), quot(0), rest(0) {
        if (pieces > 0) quot = total / pieces, rest = total - quot * pieces;
    }
    // the first `rest` pieces are one longer
    __device__ __forceinline__ int begin(int i) const { return i * quot + min(i, rest); }
    __device__ __forceinline__ int piece(int x) const {  // the piece that holds x
        const int longer = rest * (quot + 1);
        return x < longer ? x / (quot + 1) : rest + (x - longer) / quot;
    }
};

// A segment: the steps [tile0, tile1) of one triple that lie in a piece.
struct Segment {
    int seq, len, n;          // the sequence, its slots and steps
    int unit, row_begin;      // the triple of this sequence and its first place on the line
    int head, block;          // its kv head and block of rows
    int tile0, tile1, slot_end;
};

// Walks the segments of the piece [pos, end).  `units` triples share a
// sequence's length, `blocks` of them a kv head; a triple of n steps of STEP
// slots takes ROW_COST + n places.
template <int STEP> struct Walk {
    int pos, end, seq_begin, units, blocks;
    Segment s;
    static __device__ __forceinline__ int steps_of(int len) { return (len + STEP - 1) / STEP; }
    __device__ __forceinline__ int span() const { return s.n ? (s.n + ROW_COST) * units : 0; }
    __device__ __forceinline__ void length(int len) { s.len = len, s.n = steps_of(len); }
    // the segment at pos; false when the piece ends before its first step
    __device__ __forceinline__ bool enter(const PagedKv &kv) {
        while (pos >= seq_begin + span()) {  // the next sequence with slots
            seq_begin += span();
            length(paged_len(kv, ++s.seq));
        }
        s.unit = (pos - seq_begin) / (s.n + ROW_COST);
        s.head = s.unit / blocks;
        s.block = s.unit - s.head * blocks;
        s.row_begin = seq_begin + s.unit * (s.n + ROW_COST);
        s.tile0 = max(0, pos - s.row_begin - ROW_COST);
        s.tile1 = min(s.n, end - s.row_begin - ROW_COST);
        s.slot_end = min(s.len, s.tile1 * STEP);
        return s.tile0 < s.tile1;
    }
    // the next segment, if there is one
    __device__ __forceinline__ bool next(const PagedKv &kv) {
        pos = s.row_begin + ROW_COST + s.tile1;
        return pos < end && enter(kv);
    }
};

// Sums the sequences' costs and finds the one in which piece `piece` of at
// most `most` begins; false when there is nothing in it.  All THREADS threads
// of the block.
template <int THREADS, int STEP>
__device__ __forceinline__ bool find_start(const PagedKv &kv, int blocks, int piece, int most, int least, Line &line, Walk<STEP> &w) {
    constexpr int WARPS = THREADS / 32;
    __shared__ int s_warp[WARPS], s_seq, s_begin, s_len;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = kv.a.n_seqs;
    const int units = kv.a.n_kv_heads * blocks;
    // inclusive scan of the costs of sequences base .. base + THREADS - 1
    int len = 0, own = 0, incl = 0, all = 0;
    auto scan = [&](int base) {
        len = base + tid < n ? paged_len(kv, base + tid) : 0;
        own = len ? (Walk<STEP>::steps_of(len) + ROW_COST) * units : 0;
        incl = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += y;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int x = 0; x < WARPS; ++x) {
            if (x < warp) incl += s_warp[x];
            all += s_warp[x];
        }
    };
    int total = 0;
    for (int base = 0; base < n; base += THREADS) {
        scan(base);
        total += all;
    }
    // as many pieces as the GPU holds at once, or whole multiples where they stay long
    const int waves = max(1, total / (PIECE * least));
    line = Line(total, min(min(waves * least, most), total));
    if (piece >= line.pieces) return false;
    w.pos = line.begin(piece);
    w.end = line.begin(piece + 1);
    w.units = units;
    w.blocks = blocks;
    int before = 0;
    if (n <= THREADS) {
        if (incl > w.pos && incl - own <= w.pos) s_seq = tid, s_begin = incl - own, s_len = len;
    } else {
        for (int base = 0; before <= w.pos; base += THREADS) {
            scan(base);
            if (before + incl > w.pos && before + incl - own <= w.pos) s_seq = base + tid, s_begin = before + incl - own, s_len = len;
            before += all;
        }
    }
    __syncthreads();
    w.s.seq = s_seq;
    w.seq_begin = s_begin;
    w.length(s_len);
    return w.enter(kv);
}

// Infinities and NaNs among the values: a weight goes in as two 16-bit parts, of
// which the second may be zero or negative, and a row that does not see a slot
// gives it weight zero; either makes a NaN of what should be infinity or finite.
// So the steps that not every row sees count such values as zeros, and where a
// segment met one (or a row has a NaN that its weights do not explain) its values
// are looked through once more: an element that is not finite among the slots that
// a row sees becomes the sum of what is not.
enum : uint32_t { SAW_PLUS = 1, SAW_MINUS = 2, SAW_NAN = SAW_PLUS | SAW_MINUS };  // and so both infinities are a NaN

// Which of them are in 16 bits.
template <typename T> __device__ __forceinline__ uint32_t saw(uint32_t x) {
    constexpr uint32_t INF = Half16<T>::type == ABRA_GGML_F16 ? 0x7c00u : 0x7f80u;
    x &= 0xffffu;
    return (x & 0x7fffu) < INF ? 0u : (x & 0x7fffu) > INF ? SAW_NAN : x >> 15 ? SAW_MINUS : SAW_PLUS;
}
// Codes are two bits an element, 16 elements a word: element i's, where x becomes
// the sum of what is not finite.
__device__ __forceinline__ float with_saw(float x, const uint32_t *codes, int i) {
    const uint32_t seen = codes[i >> 4] >> 2 * (i & 15) & 3u;
    return seen == 0 ? x : seen == SAW_PLUS ? INFINITY : seen == SAW_MINUS ? -INFINITY : NAN;
}

// Collects in codes [row][D], zeros before, what rows r0 .. r0 + n - 1 see in
// slots [from, to); row r sees those before all_see + r / group.  All THREADS
// threads, between barriers.  One more read of the segment's values, 16 bytes a
// lane and four in flight (8 sequences of 4,096 slots with an infinity each, 64
// rows a kv head: 66 us for 31 without them; each thread's own walk of one slot
// after the other took 5,000).
template <typename T, int D, int THREADS>
__device__ __noinline__ void look_through(const AttendArgs &p, int seq, int head, int from, int to, int all_see, int r0, int n,
                                          int tid, uint32_t *codes) {
    constexpr int CH = D / 8, BATCH = 4;
    const int64_t end = static_cast<int64_t>(to - from) * CH;
    for (int64_t x0 = tid; x0 < end; x0 += BATCH * THREADS) {
        uint4 v[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int64_t x = x0 + b * THREADS;
            const int t = from + static_cast<int>(x / CH);
            v[b] = make_uint4(0, 0, 0, 0);
            if (x < end) {
                const int e = p.kv.page.div(t), page = max(0, paged_page(p.kv, seq, e));
                v[b] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.kv.a.v) +
                                                        paged_v_at(p.kv, page, head, t - e * p.kv.a.page_size) + 8 * (x % CH));
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const uint32_t w[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
            uint32_t code = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) code |= saw<T>(w[i / 2] >> 16 * (i % 2)) << 2 * i;
            if (code == 0) continue;
            const int64_t x = x0 + b * THREADS;
            const int t = from + static_cast<int>(x / CH), chunk = static_cast<int>(x % CH);
            code <<= 16 * (chunk % 2);
            const int64_t first = static_cast<int64_t>(t - all_see + 1) * p.group - r0;  // the first row that sees it
            for (int r = static_cast<int>(max(static_cast<int64_t>(0), first)); r < n; ++r) {
                uint32_t *at = codes + r * (D / 16) + chunk / 2;
                if (code & ~*reinterpret_cast<volatile uint32_t *>(at)) atomicOr(at, code);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_out(const AttendArgs &p, int64_t at, float4 x) {
    if (p.out_f32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = x;
    } else {
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + at) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    }
}

// log2 of a row's sum of 2^s.
template <typename T> __device__ __forceinline__ float row_lse2(float m, float total) {
    return total != 0.0f ? m + log2f(total * power_of_two(-Weigh<T>::SHIFT)) : -INFINITY;
}

// A finished row's lse; total == 0: the row saw nothing.
template <typename T>
__device__ __forceinline__ void finish_lse(const AttendArgs &p, int seq, int head, int r, float m, float total) {
    const int j = r / p.group, h = head * p.group + r - j * p.group;
    const float l2 = row_lse2<T>(m, total);
    if (p.lse) p.lse[(static_cast<int64_t>(seq) * p.n_q + j) * p.n_heads + h] = l2 * 0.69314718055994531f;
    if (p.row_lse) p.row_lse[(static_cast<int64_t>(seq) * p.kv.a.n_kv_heads + head) * p.rows + r] = l2;
}

// A finished row: out at elements d .. d + 3, its lse by the lane of element 0.
template <typename T>
__device__ __forceinline__ void finish_row(const AttendArgs &p, int seq, int head, int r, int d, int D, float4 o, float m,
                                           float total) {
    const int j = r / p.group, h = head * p.group + r - j * p.group;
    const int64_t row = static_cast<int64_t>(seq) * p.n_q + j;
    const float inv = total != 0.0f ? 1.0f / total : 0.0f;
    store_out<T>(p, row * p.ldo + static_cast<int64_t>(h) * D + d,
                 total != 0.0f ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0, 0, 0, 0));
    if (d == 0) finish_lse<T>(p, seq, head, r, m, total);
}

// The kernel for blocks of 16 to 64 rows (paged_attention_wide.cu); one CTA a
// multiprocessor.  `n`: rows of a block, 16, 32 or 64.
constexpr int WIDE_STEP = 128;  // its slots a step
cudaError_t launch_attend_wide(const AttendArgs &p, int n, int pieces, bool scores, cudaStream_t st);

}  // namespace abra
