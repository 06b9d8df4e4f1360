// kv4_attn.cu -- attention of one query a sequence over the paged 4-bit cache
// (holo_b200.h, cuda_kv4_attention).
//
// Bound by the read of the cache, 18 bytes for 32 values; the work per byte is
// the codes' conversion, so it is kept to a few instructions a word of eight:
//   scores   A word of key codes, masked, is two fp16 subnormals n * 2^-24 (or,
//            four bits up, 16 n * 2^-24): exact operands of mma.m16n8k16
//            without a conversion (A: 16 positions, B: 8 query heads).  q is
//            laid out to match, the 16 taken out of it; the accumulator of
//            each group of 32 starts at -8 * 2^-24 * sum(q), which makes the codes
//            signed, and its result is multiplied by the group's scale.
//   values   A pair of codes is taken from two positions' words, and is an fp16
//            operand the same way; A: 16 dims, B: the softmax weights of 8 heads
//            times the position's scale of the group, transposed by movmatrix.
//            One more MMA with A all -8 * 2^-24 makes the codes signed 16
//            positions at a time, before the sum could grow by them.
// Only the weights are rounded, to fp16.  So that they use fp16's range whatever
// the values' size, they are scaled by a power of two that follows the largest
// scale seen; a head's q is scaled by the power of two of its largest value.
//   fp32 rows  q and the weights have a second fp16 term that carries the rest.
//            The tensor core lines products up by their operands' exponents, a
//            subnormal's being 2^-14 whatever it holds, and drops what falls below: a sum of
//            subnormals keeps 2^-18 of itself.  That is enough for rows of 16
//            bits and not here, so the codes become normal numbers n - 8, an
//            instruction more an operand but no MMA for the signs; and as its sums are
//            cut towards 0, a block's sum of values is added to the others outside of it.
//
// The units of work, 64 positions of 8 heads of one KV head, of all sequences form one
// list that is cut evenly over the CTAs (ragged batches stay balanced).  Each warp
// streams every fourth unit of its CTA's part through a ring of its own, one
// bulk copy a block of 16 positions, its table entry loaded a unit ahead, and
// keeps a running maximum, sum and output; warps join in shared memory.  A
// list item that is cut leaves partial results, and the CTA that comes last joins them in
// their order, so the result does not depend on timing; items of up to AT_WHOLE
// units are not cut, so that a short sequence's result does not depend on its batch either.
//
// Measured: bound by instruction issue and, in long runs, by the board's power.  A unit takes a
// warp 3500 cycles with two warps a scheduler (two CTAs an SM at 128 dims;
// 12 warps an SM in three CTAs of 32-position units: 59.6 us against 61.7 in the batch below, but
// 14.0 against 11.8 for one sequence and 164 against 157 for the long ones).  64 sequences
// of up to 4096 (64 heads over 8 of 128, fp16): 55.7 us, 3.0 TB/s; 8 of up to
// 131072 (bf16): 154 to 166 us, 4.0 to 4.3 TB/s; one of 2047 (32 over 32, fp32): 11.7 us, of which launch,
// cut, tables and joins are 8.  9 to 16 heads a KV head are two items, each of which reads and
// unpacks the cache: 111 us for 64 sequences with 128 heads over 8 (58 with 64 of the same lengths' range).  Head
// size 256 has room for one CTA an SM: 135 us, and in fp32, where it spills (152 bytes of stores a thread), 275.
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int AT_WARPS = 4, AT_THREADS = 32 * AT_WARPS;
constexpr int AT_UNIT = 4;                     // blocks of 16 positions a unit
constexpr int AT_UNIT_POS = AT_UNIT * KV4_BLOCK;
constexpr int AT_WHOLE = 8;                    // items of up to so many units are not cut
constexpr int AT_MIN = 4;                      // units a CTA: fewer cost more to join than they save
constexpr int AT_ITEM = 4;                     // the cost of an item where CTAs take several
constexpr float AT_GROWTH = 6.0f;              // log2 of what a maximum may grow by before the sums are rescaled
constexpr int AT_SHIFT = 8;                    // weights times scales lie below 2 to this and AT_GROWTH: 2^14

template <int HD> struct AtGeom {
    static constexpr int NB = HD / KV4_GROUP;
    static constexpr int BLOCK_BYTES = kv4_block_bytes(HD);
    static constexpr int STAGES = HD == 64 ? 3 : 2;
    static constexpr int RING = AT_WARPS * STAGES * AT_UNIT * BLOCK_BYTES;
    static constexpr int ROW = HD + 4;          // floats of a head in the join: its lanes' 16-byte stores spread over all banks
    static constexpr int JOIN = AT_WARPS * KV4_HEADS * ROW * 4;
    static constexpr int SMEM = RING + JOIN;
    static constexpr int CTAS = HD == 256 ? 1 : HD == 128 ? 2 : 3;   // an SM
    static constexpr int SLOT = KV4_HEADS * (HD + 2);   // floats of a partial result: m and l of the heads, then the outputs
};

struct AtArgs {
    void *out;
    const void *q;
    long long q_row, out_row;
    const int *seqs;
    int n, n_heads, group, chunks;             // chunks of KV4_HEADS query heads a KV head
    int item_cost;                             // what an item costs besides its units, in units: its q, the join
    float scale;
    uint32_t page_magic;                       // ceil(2^32 / page_blocks); 0 for 1
    bool wide, q_wide;                         // rows of out, and of q, are 16-byte aligned
    int *counters;
    float *partial;
};

__device__ __forceinline__ float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// d = a b + c: pure, so that the compiler may interleave independent ones
__device__ __forceinline__ void at_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void at_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t at_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t at_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 at_unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
// Codes n and their fp16 operands.  Plain: the subnormals n 2^-24, by a mask.
// Signed: n - 8, an exponent set beside the code and taken off again.  Of odd codes, 16 times these.
constexpr uint32_t AT_EVEN = 0x000f000fu, AT_ODD = 0x00f000f0u;
template <uint32_t CODES, bool SIGNED> __device__ __forceinline__ uint32_t at_codes(uint32_t w) {
    if (!SIGNED) return w & CODES;
    const uint32_t x = (w & CODES) | 0x64006400u;   // 1024 + n; 1024 + 16 n
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&x), __float2half2_rn(CODES == AT_EVEN ? 1032.0f : 1152.0f));
    return *reinterpret_cast<const uint32_t *>(&y);
}
template <int N> struct AtWords { uint32_t w[N]; };
template <int N> __device__ __forceinline__ AtWords<N> at_lds(const uint8_t *p) {
    AtWords<N> r;
    if constexpr (N == 1) r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    else if constexpr (N == 2) *reinterpret_cast<uint2 *>(r.w) = *reinterpret_cast<const uint2 *>(p);
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4 *>(r.w + i) = *reinterpret_cast<const uint4 *>(p + 4 * i);
    }
    return r;
}

// The list: of every sequence, every (KV head, chunk of heads), its units after
// item_cost places that stand for the rest of its work.  A walk through the CTA's
// part, item by item.
struct Walk {
    int i, s, len, units;      // sequence: its place in the list, number, positions, units an item
    int item;                  // KV head * chunks + chunk
    int start;                 // of the item in the list
    uint32_t number;           // counts the items in which the warp has units
    int first, take;           // its units in the part
};

__device__ __forceinline__ int at_units(const Kv4View &c, const AtArgs &a, int i, int &s, int &len) {
    s = a.seqs ? __ldcg(a.seqs + i) : i;
    len = 0;
    if (s < 0 || s >= c.max_seqs) {
        s = -1;
        return 0;
    }
    len = max(0, min(__ldcg(c.lens + s), c.max_pages * c.page_tokens));
    return (len + AT_UNIT_POS - 1) / AT_UNIT_POS;
}
// the item's units in [from, to) of the list
__device__ __forceinline__ void at_clip(const AtArgs &a, Walk &w, int from, int to) {
    w.first = max(0, from - w.start - a.item_cost);
    w.take = max(0, min(w.units, to - w.start - a.item_cost) - w.first);
}
// the next item of the part [from, to) that has units in it; false: none.  unit0: the warp's first one of an item's
__device__ __forceinline__ bool at_next(const Kv4View &c, const AtArgs &a, Walk &w, int from, int to, int unit0) {
    do {
        w.start += w.units + a.item_cost;
        w.first = w.take = 0;
        if (w.start >= to) return false;
        if (++w.item == c.n_kv * a.chunks) {
            w.item = 0;
            do {
                if (++w.i >= a.n) return false;
                w.units = at_units(c, a, w.i, w.s, w.len);
            } while (w.units == 0);
        }
        at_clip(a, w, from, to);
    } while (w.take == 0);
    w.number += w.take > unit0;
    return true;
}

// inclusive sum over the CTA
__device__ __forceinline__ int at_scan(int v, int *sh, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) {
        if (w < warp) v += sh[w];
        total += sh[w];
    }
    return v;
}

// the values of q that a lane holds, as they lie: eight of every group
template <typename T, int NB> struct AtQ {
    alignas(16) T v[NB][8];
    __device__ __forceinline__ void load(const T *q, bool wide, bool there) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; e += N) {
                if (!there) *reinterpret_cast<uint4 *>(&v[b][e]) = make_uint4(0, 0, 0, 0);
                else if (wide) *reinterpret_cast<uint4 *>(&v[b][e]) = __ldcg(reinterpret_cast<const uint4 *>(q + 32 * b + e));
                else
#pragma unroll
                    for (int i = 0; i < N; ++i) v[b][e + i] = q[32 * b + e + i];
            }
    }
};

template <typename T>
__device__ __forceinline__ void at_store4(T *p, bool wide, float x, float y, float z, float w) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
        } else {
            uint2 u;
            T *h = reinterpret_cast<T *>(&u);
            h[0] = kv4_from_float<T>(x), h[1] = kv4_from_float<T>(y), h[2] = kv4_from_float<T>(z), h[3] = kv4_from_float<T>(w);
            *reinterpret_cast<uint2 *>(p) = u;
        }
    } else {
        p[0] = kv4_from_float<T>(x), p[1] = kv4_from_float<T>(y), p[2] = kv4_from_float<T>(z), p[3] = kv4_from_float<T>(w);
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(AT_THREADS, AtGeom<HD>::CTAS)
kv4_attn_kernel(const __grid_constant__ Kv4View c, const __grid_constant__ AtArgs a) {
    using G = AtGeom<HD>;
    constexpr int NB = G::NB, STAGES = G::STAGES;
    constexpr bool FINE = sizeof(T) == 4;      // fp32 rows: second terms of q and of the weights
    constexpr int TERMS = FINE ? 2 : 1;
    constexpr float UNIT = FINE ? 1.0f : 16777216.0f;   // 1 / a code's operand
    extern __shared__ __align__(128) uint8_t at_smem[];
    __shared__ uint64_t full[AT_WARPS][STAGES];
    __shared__ int scan[AT_WARPS];
    __shared__ Walk begin;
    __shared__ int part_start, part_end;
    __shared__ float join_m[AT_WARPS][KV4_HEADS], join_l[AT_WARPS][KV4_HEADS], join_w[AT_WARPS][KV4_HEADS];
    __shared__ float join_den[KV4_HEADS];
    __shared__ int last;
    // Items (a bit each, by their number: no more than the ring's slots are under way) of which the warp met a table entry that
    // names no page.  Such an item comes out as zeros: its share's sum of weights is given as -1, which no sum of
    // exponentials is, up to the last join.
    __shared__ uint32_t bad_items[AT_WARPS];
    float *join = reinterpret_cast<float *>(at_smem + G::RING);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t *ring = at_smem + (size_t)warp * STAGES * AT_UNIT * G::BLOCK_BYTES;

    if (lane < STAGES) mbar_init(&full[warp][lane], 1);
    if (lane == 0) bad_items[warp] = 0;
    fence_barrier_init();
    early_wait();
    early_next();

    bool empty = false;                       // there are sequences without positions
    auto zeros = [&]() {                      // theirs (a number out of range: left alone)
        if (!empty) return;
        for (int i = blockIdx.x; i < a.n; i += gridDim.x) {
            int s, len;
            if (at_units(c, a, i, s, len) == 0 && s >= 0)
                for (int d = 4 * threadIdx.x; d < a.n_heads * HD; d += 4 * AT_THREADS)
                    at_store4<T>((T *)a.out + i * a.out_row + d, a.wide, 0.0f, 0.0f, 0.0f, 0.0f);
        }
    };

    // ---- the CTA's part of the list ----
    const int items = c.n_kv * a.chunks;
    int all = 0, held = 0, s0 = -1, len0 = 0, u0 = 0, end0 = 0;   // s0 .. end0: of the thread's sequence in the last step
    auto places = [&](int units) { return units ? (units + a.item_cost) * items : 0; };
    for (int i0 = 0; i0 < a.n; i0 += AT_THREADS) {
        const int i = i0 + threadIdx.x;
        u0 = 0, s0 = -1, len0 = 0;
        if (i < a.n) {
            u0 = at_units(c, a, i, s0, len0);
            if (s0 < 0 && blockIdx.x == 0) kv4_report(c.status, HOLO_E_ARG);
        }
        int total;
        end0 = all + at_scan(places(u0), scan, total);
        all += total;
        held += __syncthreads_count(u0 > 0);
    }
    empty = held < a.n;
    // a CTA an item, or more where they keep AT_MIN units each
    const int units = all - held * items * a.item_cost;
    const int ctas = max(1, min(min((int)gridDim.x, units), max(held * items, units / AT_MIN)));
    if ((int)blockIdx.x >= ctas) {
        zeros();
        return;
    }
    // Its part: `step` places of the list, the cuts moved down to the item's start
    // where the item is short.  Cuts inside longer items stay, so that the parts that an item spans follow from them.
    const int step = (all + ctas - 1) / ctas;
    const int cut0 = (int)blockIdx.x * step, cut1 = min(all, cut0 + step);
    if (cut0 >= all) {                        // rounded up, they took all of it
        zeros();
        return;
    }
    if (threadIdx.x == 0) part_start = 0, part_end = cut1 == all ? all : 0;
    __syncthreads();
    {
        int before = 0;
        for (int i0 = 0; i0 < a.n && before <= cut1; i0 += AT_THREADS) {
            if (a.n > AT_THREADS) {           // else as the sum left it
                const int i = i0 + threadIdx.x;
                u0 = 0, s0 = -1, len0 = 0;
                if (i < a.n) u0 = at_units(c, a, i, s0, len0);
                int total;
                end0 = before + at_scan(places(u0), scan, total);
                before += total;
            }
            const int start = end0 - places(u0), item_places = u0 + a.item_cost;
            if (start <= cut0 && cut0 < end0) {
                Walk w;
                w.i = i0 + threadIdx.x, w.s = s0, w.len = len0, w.units = u0;
                w.item = (cut0 - start) / item_places;
                w.start = start + w.item * item_places;
                w.number = 0;
                begin = w;
                part_start = u0 > AT_WHOLE ? cut0 : w.start;
            }
            if (start <= cut1 && cut1 < end0)
                part_end = u0 > AT_WHOLE ? cut1 : start + (cut1 - start) / item_places * item_places;
        }
        __syncthreads();
    }
    int from = part_start, to = part_end;
    // Where every item is one unit and the part has several, each warp takes a quarter of them
    // for itself, and nothing is joined (the join of one warp's result leaves it as it is): 96
    // sequences of up to 60, 32 heads of 128 over 32, in 20.8 us and not 47.2; a single item is no sooner done.
    const int unit_items = units == held * items ? (to - from) / (1 + a.item_cost) : 0;
    const bool solo = unit_items > 1;
    if (solo) {
        to = from + unit_items * (warp + 1) / AT_WARPS * (1 + a.item_cost);
        from += unit_items * warp / AT_WARPS * (1 + a.item_cost);
    }
    const int unit0 = solo ? 0 : warp, unit_step = solo ? 1 : AT_WARPS;
    Walk head = begin;
    bool any = from < to;
    if (any) {
        at_clip(a, head, from, to);
        if (head.take == 0) any = at_next(c, a, head, from, to, unit0);
    }
    if (!any) {
        zeros();
        return;
    }

    // q of head g of an item's, quarter t of every group: loaded before it is wanted
    AtQ<T, NB> raw;
    auto heads_of = [&](const Walk &x, int &first) {
        const int kvh = x.item / a.chunks;
        first = kvh * a.group + (x.item % a.chunks) * KV4_HEADS;
        return min(KV4_HEADS, (kvh + 1) * a.group - first);
    };
    auto load_q = [&](const Walk &x) {
        int first;
        const int n = heads_of(x, first);
        raw.load((const T *)a.q + x.i * a.q_row + (long long)(first + g) * HD + 8 * t, a.q_wide, g < n);
    };
    constexpr bool EARLY = HD < 256;          // else its registers would be spilled
    // ---- the warp's loads: unit `unit` of item `load` ----
    // The walks lie in shared memory (one a warp each): only an item's change reads them.
    __shared__ Walk walk_load[AT_WARPS], walk_use[AT_WARPS];
    Walk &load = walk_load[warp], &w = walk_use[warp];
    if (lane == 0) load = head, w = head;
    __syncwarp();
    int unit = head.first + unit0, unit_end, load_len;   // unit_end 0: no more
    const uint8_t *load_base;                 // of the KV head
    const int *load_table;
    const uint32_t page_bytes = (uint32_t)c.n_kv * c.page_blocks * G::BLOCK_BYTES;
    auto settle = [&]() {                     // to the next unit that there is, and its item
        Walk x = load;
        bool more = true;
        while (more && unit >= x.first + x.take) {
            more = at_next(c, a, x, from, to, unit0);
            unit = x.first + unit0;
        }
        __syncwarp();
        if (lane == 0) load = x;
        __syncwarp();
        unit_end = more ? x.first + x.take : 0;
        load_len = x.len;
        load_base = c.pool + (uint32_t)(x.item / a.chunks * c.page_blocks * G::BLOCK_BYTES);
        load_table = c.tables + (size_t)max(0, x.s) * c.max_pages;
    };
    settle();
    int entry = -1, in_page = 0;              // the first lanes: the page of their block of it, and the block there
    auto look_up = [&]() {
        const int block = unit * AT_UNIT + lane;
        if (unit < unit_end && lane < AT_UNIT && block * KV4_BLOCK < load_len) {
            const int col = a.page_magic ? (int)__umulhi((uint32_t)block, a.page_magic) : block;
            in_page = block - col * c.page_blocks;
            entry = __ldcg(load_table + col);
        }
    };
    look_up();
    if (EARLY) load_q(head);
    int ahead = 0, fill = 0;                  // units issued and not yet taken, the slot of the next one
    auto issue = [&]() {                      // its copies, and the table entries of the next one
        if (unit >= unit_end) return;
        const int blocks = min(AT_UNIT, (load_len - unit * AT_UNIT_POS + KV4_BLOCK - 1) / KV4_BLOCK);
        if (lane == 0) mbar_arrive_expect_tx(&full[warp][fill], blocks * G::BLOCK_BYTES);
        __syncwarp();
        if (lane < blocks) {
            if ((uint32_t)entry >= (uint32_t)c.n_pages) {   // any page, so that the ring goes on: the item's result is dropped
                kv4_report(c.status, HOLO_E_ARG);
                atomicOr(&bad_items[warp], 1u << (load.number & 31));
                entry = 0;
            }
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                :: "r"(smem_addr(ring + (fill * AT_UNIT + lane) * G::BLOCK_BYTES)),
                   "l"(load_base + (size_t)(uint32_t)entry * page_bytes + in_page * G::BLOCK_BYTES), "r"(G::BLOCK_BYTES),
                   "r"(smem_addr(&full[warp][fill])) : "memory");
        }
        ++ahead;
        fill = fill + 1 == STAGES ? 0 : fill + 1;
        unit += unit_step;
        if (unit >= unit_end) settle();
        look_up();
    };
    __syncwarp();
    issue();                                  // the others when q has been laid out: their table entries are on the way

    // ---- items ----
    int slot = 0, phase = 0;                  // the slot of the next unit to take and its barrier's phase
    bool ok = true;
    for (bool more = true, begun = false; more; begun = true) {
        const int len = w.len, u_end = w.first + w.take;
        int head0;
        const int heads = heads_of(w, head0);
        if (!EARLY) load_q(w);
        // q, times a power of two; B fragments of the two steps of a group
        uint32_t qf[TERMS][NB][2][2];
        float start[NB][2], factor[2];        // of heads 2 t and 2 t + 1
        {
            float qv[NB][8], top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    qv[b][e] = kv4_to_float<T>(raw.v[b][e]);
                    top = fmaxf(top, fabsf(qv[b][e]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(11 - exponent) brings the largest to [2^11, 2^12)
            const int e0 = max(12, (int)(__float_as_uint(top) >> 23));
            const float up = __uint_as_float((uint32_t)(265 - e0) << 23);
            // (never 0, which would make NaN of a masked score)
            const float down = fmaxf(__uint_as_float((uint32_t)(e0 - 11) << 23) * a.scale * 1.4426950408889634f * UNIT, 1.17549435e-38f);
            float sum[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                sum[b] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // codes e and e + 4 share a register; odd ones are 16 times as large
                    const float x = qv[b][e] * up, y = qv[b][e + 4] * up, odd = e & 1 ? 0.0625f : 1.0f;
                    uint32_t f = at_pack(x * odd, y * odd);
                    qf[0][b][e & 1][e >> 1] = f;
                    float2 r = at_unpack(f);
                    float sx = r.x, sy = r.y;
                    if (FINE) {
                        f = at_pack(x * odd - r.x, y * odd - r.y);
                        qf[TERMS - 1][b][e & 1][e >> 1] = f;
                        r = at_unpack(f);
                        sx += r.x, sy += r.y;
                    }
                    sum[b] += (sx + sy) * (e & 1 ? 16.0f : 1.0f);
                }
                sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
                sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
                sum[b] *= -8.0f / 16777216.0f;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int from = 4 * (2 * t + x);
                factor[x] = __shfl_sync(0xffffffffu, down, from);
#pragma unroll
                for (int b = 0; b < NB; ++b) start[b][x] = __shfl_sync(0xffffffffu, sum[b], from);
            }
        }
        float o[NB][2][4];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][x][e] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        int power = -32;                      // of two: the largest |value scale| lies below it

        if (!begun)
            for (int k = 1; k < STAGES; ++k) issue();
        for (int u = w.first + unit0; u < u_end; u += unit_step) {
            ok = ok && mbar_wait_bounded(&full[warp][slot], phase, c.status, HOLO_E_TIMEOUT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint8_t *buf = ring + slot * AT_UNIT * G::BLOCK_BYTES;
            --ahead;
            if (++slot == STAGES) slot = 0, phase ^= 1;
            const int left = len - u * AT_UNIT_POS;   // positions of the sequence from the unit's first on
            const bool tail = left < AT_UNIT_POS;
            // scores of positions g, g + 8 (+ 16 a block), heads 2 t and 2 t + 1
            float s[AT_UNIT][4];
            AtWords<NB / 2> dv[AT_UNIT][2];
            __half2 dmax = __float2half2_rn(0.0f);
#pragma unroll
            for (int k = 0; k < AT_UNIT; ++k) {
                const uint8_t *blk = buf + k * G::BLOCK_BYTES;
                const AtWords<NB> w0 = at_lds<NB>(blk + g * (HD / 2) + t * 4 * NB);
                const AtWords<NB> w1 = at_lds<NB>(blk + (g + 8) * (HD / 2) + t * 4 * NB);
                const AtWords<NB / 2> d0 = at_lds<NB / 2>(blk + kv4_off_dk(HD) + g * 2 * NB);
                const AtWords<NB / 2> d1 = at_lds<NB / 2>(blk + kv4_off_dk(HD) + (g + 8) * 2 * NB);
                dv[k][0] = at_lds<NB / 2>(blk + kv4_off_dv(HD) + g * 2 * NB);
                dv[k][1] = at_lds<NB / 2>(blk + kv4_off_dv(HD) + (g + 8) * 2 * NB);
                float acc[NB][4];
                if (!FINE) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        at_mma(acc[b], w0.w[b] & AT_EVEN, w1.w[b] & AT_EVEN, w0.w[b] >> 8 & AT_EVEN, w1.w[b] >> 8 & AT_EVEN,
                               qf[0][b][0][0], qf[0][b][0][1], start[b][0], start[b][1], start[b][0], start[b][1]);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        at_mma(acc[b], w0.w[b] & AT_ODD, w1.w[b] & AT_ODD, w0.w[b] >> 8 & AT_ODD, w1.w[b] >> 8 & AT_ODD,
                               qf[0][b][1][0], qf[0][b][1][1]);
                } else {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t w[4] = {w0.w[b], w1.w[b], w0.w[b] >> 8, w1.w[b] >> 8};
                        uint32_t even[4], odd[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) even[i] = at_codes<AT_EVEN, FINE>(w[i]), odd[i] = at_codes<AT_ODD, FINE>(w[i]);
#pragma unroll
                        for (int f = TERMS - 1; f >= 0; --f) {
                            if (f == TERMS - 1)
                                at_mma(acc[b], even[0], even[1], even[2], even[3], qf[f][b][0][0], qf[f][b][0][1], 0.0f, 0.0f, 0.0f, 0.0f);
                            else at_mma(acc[b], even[0], even[1], even[2], even[3], qf[f][b][0][0], qf[f][b][0][1]);
                            at_mma(acc[b], odd[0], odd[1], odd[2], odd[3], qf[f][b][1][0], qf[f][b][1][1]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[k][e] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float2 e0 = at_unpack(d0.w[b >> 1]), e1 = at_unpack(d1.w[b >> 1]);
                    const float s0 = b & 1 ? e0.y : e0.x, s1 = b & 1 ? e1.y : e1.x;
                    s[k][0] = fmaf(s0, acc[b][0], s[k][0]);
                    s[k][1] = fmaf(s0, acc[b][1], s[k][1]);
                    s[k][2] = fmaf(s1, acc[b][2], s[k][2]);
                    s[k][3] = fmaf(s1, acc[b][3], s[k][3]);
                }
                if (tail) {                   // past the end: weight 0, whatever lies there
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (16 * k + g + 8 * x >= left) {
                            s[k][2 * x] = s[k][2 * x + 1] = -INFINITY;
#pragma unroll
                            for (int i = 0; i < NB / 2; ++i) dv[k][x].w[i] = 0;
                        }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i)
                        dmax = __hmax2(dmax, __habs2(*reinterpret_cast<const __half2 *>(&dv[k][x].w[i])));
            }
            // Maxima of the lane's positions, and of the scales.  Only where one has grown by more than
            // AT_GROWTH (a scale: by a power of two) is the warp's maximum taken and the sums rescaled.
            float mn[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mn[x] = fmaxf(s[0][x], s[0][x + 2]);
#pragma unroll
                for (int k = 1; k < AT_UNIT; ++k) mn[x] = fmaxf(mn[x], fmaxf(s[k][x], s[k][x + 2]));
                mn[x] *= factor[x];
            }
            const uint32_t big = (uint32_t)__half_as_ushort(__hmax(__low2half(dmax), __high2half(dmax)));
            if (__any_sync(0xffffffffu, mn[0] > m[0] + AT_GROWTH || mn[1] > m[1] + AT_GROWTH || (int)(big >> 10) - 14 > power)) {
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) {
                    mn[0] = fmaxf(mn[0], __shfl_xor_sync(0xffffffffu, mn[0], i));
                    mn[1] = fmaxf(mn[1], __shfl_xor_sync(0xffffffffu, mn[1], i));
                }
                // fp16 exponent field e: below 2^(e - 14)
                const int pn = max(power, (int)(__reduce_max_sync(0xffffffffu, big) >> 10) - 14);
                const float lower = __uint_as_float((uint32_t)(127 + power - pn) << 23);   // 2^(power - pn)
                float fix[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mn[x] = fmaxf(ceilf(mn[x]), m[x]);   // whole: rescaling is exact
                    fix[x] = (mn[x] > m[x] ? at_ex2(m[x] - mn[x]) : 1.0f) * lower;
                    l[x] *= fix[x];
                    m[x] = mn[x];
                }
                power = pn;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[b][x][e] *= fix[e & 1];
            }
            // weights 2^(s - m) times 2^(AT_SHIFT - power)
            float sub[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) sub[x] = (m[x] == -INFINITY ? 0.0f : m[x]) + (float)(power - AT_SHIFT);
#pragma unroll
            for (int k = 0; k < AT_UNIT; ++k) {
                const uint8_t *blk = buf + k * G::BLOCK_BYTES;
                if (16 * k >= left) break;    // a block that was not loaded
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = at_ex2(fmaf(s[k][e], factor[e & 1], -sub[e & 1]));
                    l[e & 1] += p[e];
                }
                // codes of positions 2 t, 2 t + 1 and 2 t + 8, 2 t + 9, values 4 g .. 4 g + 3 of every group
                const uint8_t *v = blk + kv4_off_v(HD) + ((g >> 1) * 8 * 2 + (g & 1)) * 4 * NB;
                const AtWords<NB> v0 = at_lds<NB>(v + t * 8 * NB), v1 = at_lds<NB>(v + (t + 4) * 8 * NB);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float2 e0 = at_unpack(dv[k][0].w[b >> 1]), e1 = at_unpack(dv[k][1].w[b >> 1]);
                    const float s0 = b & 1 ? e0.y : e0.x, s1 = b & 1 ? e1.y : e1.x;
                    float y[4] = {p[0] * s0, p[1] * s0, p[2] * s1, p[3] * s1};
                    uint32_t pf[TERMS][2];
#pragma unroll
                    for (int f = 0; f < TERMS; ++f) {
                        const uint32_t lo = at_pack(y[0], y[1]), hi = at_pack(y[2], y[3]);
                        pf[f][0] = at_transpose(lo);
                        pf[f][1] = at_transpose(hi);
                        if (f + 1 < TERMS) {
                            const float2 a0 = at_unpack(lo), a1 = at_unpack(hi);
                            y[0] -= a0.x, y[1] -= a0.y, y[2] -= a1.x, y[3] -= a1.y;
                        }
                    }
                    const uint32_t pick = b & 1 ? 0x7632u : 0x5410u;
                    const uint32_t x0 = __byte_perm(v0.w[b >> 1], v0.w[NB / 2 + (b >> 1)], pick);
                    const uint32_t x1 = __byte_perm(v1.w[b >> 1], v1.w[NB / 2 + (b >> 1)], pick);
                    // rows g and g + 8: codes 2 x and, 16 times as large, 2 x + 1; then -8 of each
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t c[4] = {at_codes<AT_EVEN, FINE>(x0 >> (8 * x)), at_codes<AT_ODD, FINE>(x0 >> (8 * x)),
                                               at_codes<AT_EVEN, FINE>(x1 >> (8 * x)), at_codes<AT_ODD, FINE>(x1 >> (8 * x))};
                        if (!FINE) {
                            at_mma(o[b][x], c[0], c[1], c[2], c[3], pf[0][0], pf[0][1]);
                            at_mma(o[b][x], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pf[0][0], pf[0][1]);
                        } else {      // a block's sum, added with rounding
                            float part[4];
                            at_mma(part, c[0], c[1], c[2], c[3], pf[TERMS - 1][0], pf[TERMS - 1][1], 0.0f, 0.0f, 0.0f, 0.0f);
                            at_mma(part, c[0], c[1], c[2], c[3], pf[0][0], pf[0][1]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[b][x][i] += part[i];
                        }
                    }
                }
            }
            __syncwarp();                     // the slot has been read
            issue();
        }

        // the next item (mostly where the loads are), and its q under way while the warps join
        Walk after = load;
        more = true;
        if (after.take == 0 || after.start != w.start + w.units + a.item_cost) {
            after = w;
            more = at_next(c, a, after, from, to, unit0);
        }
        if (EARLY && more) load_q(after);
        T *out = (T *)a.out + w.i * a.out_row + (long long)head0 * HD;

        // ---- join the warps ----
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], i);
        if (bad_items[warp] >> (w.number & 31) & 1) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b][x][e] = 0.0f;
            m[0] = m[1] = 0.0f;
            l[0] = l[1] = solo ? 1.0f : -1.0f;
            __syncwarp();
            if (lane == 0) bad_items[warp] &= ~(1u << (w.number & 31));
            __syncwarp();
        }
        // l and o hold 2^(AT_SHIFT - power) too; o's codes 1 / UNIT, odd ones 16 times as large
        if (solo) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (2 * t + e < heads)
                        at_store4<T>(out + (2 * t + e) * HD + 32 * b + 4 * g, a.wide, o[b][0][e] * UNIT / l[e],
                                     o[b][0][e + 2] * (UNIT / 16) / l[e], o[b][1][e] * UNIT / l[e],
                                     o[b][1][e + 2] * (UNIT / 16) / l[e]);
            __syncwarp();
            if (lane == 0) w = after;
            __syncwarp();
            continue;
        }
        const float scaled = (float)(AT_SHIFT - power);
        if (g == 0) {
            join_m[warp][2 * t] = m[0] - scaled, join_m[warp][2 * t + 1] = m[1] - scaled;
            join_l[warp][2 * t] = l[0], join_l[warp][2 * t + 1] = l[1];
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e)       // values 32 b + 4 g .. + 3 of head 2 t + e
                *reinterpret_cast<float4 *>(join + (warp * KV4_HEADS + 2 * t + e) * G::ROW + 32 * b + 4 * g) =
                    make_float4(o[b][0][e] * UNIT, o[b][0][e + 2] * (UNIT / 16), o[b][1][e] * UNIT, o[b][1][e + 2] * (UNIT / 16));
        __syncthreads();
        const bool whole = w.first == 0 && w.take == w.units;
        float *mine = a.partial + ((size_t)blockIdx.x * 2 + (w.first > 0 ? 0 : 1)) * G::SLOT;
        if (threadIdx.x < KV4_HEADS) {
            const int h = threadIdx.x;
            float top = -INFINITY, den = 0.0f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < AT_WARPS; ++i) {
                if (join_l[i][h] != 0.0f) top = fmaxf(top, join_m[i][h]);
                bad |= join_l[i][h] < 0.0f;
            }
#pragma unroll
            for (int i = 0; i < AT_WARPS; ++i) {
                const float f = join_l[i][h] != 0.0f ? at_ex2(join_m[i][h] - top) : 0.0f;
                join_w[i][h] = f;
                den = fmaf(join_l[i][h], f, den);
            }
            if (bad) den = -1.0f;
            join_den[h] = den;
            if (!whole) mine[2 * h] = top, mine[2 * h + 1] = den;
        }
        __syncthreads();
        for (int d = 4 * threadIdx.x; d < heads * HD; d += 4 * AT_THREADS) {
            const int h = d / HD;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < AT_WARPS; ++i) {
                const float4 v = *reinterpret_cast<const float4 *>(join + (i * KV4_HEADS + h) * G::ROW + d % HD);
                const float f = join_w[i][h];
                sum.x = fmaf(v.x, f, sum.x), sum.y = fmaf(v.y, f, sum.y), sum.z = fmaf(v.z, f, sum.z), sum.w = fmaf(v.w, f, sum.w);
            }
            if (whole) {
                const float den = join_den[h];
                if (den < 0.0f) at_store4<T>(out + d, a.wide, 0.0f, 0.0f, 0.0f, 0.0f);
                else at_store4<T>(out + d, a.wide, sum.x / den, sum.y / den, sum.z / den, sum.w / den);
            } else {
                *reinterpret_cast<float4 *>(mine + 2 * KV4_HEADS + d) = sum;
            }
        }
        if (!whole) {
            // The item's units lie in parts p0 .. p1; the last part to come joins their results, in order.  (A part that gave up
            // waiting comes too, so the counter is 0 after every call.)
            const int begins = w.start + a.item_cost;
            const int p0 = begins / step, p1 = (begins + w.units - 1) / step;
            int *counter = a.counters + (size_t)w.i * items + w.item;
            __syncthreads();
            if (threadIdx.x == 0) {           // of all the CTA's writes, and before its reads
                __threadfence();
                last = atomicAdd(counter, 1) == p1 - p0;
                if (last) {
                    __threadfence();
                    *counter = 0;             // for the next call
                }
            }
            __syncthreads();
            if (last) {
                const float *part = a.partial + ((size_t)p0 * 2 + 1) * G::SLOT;   // then every second one, one less
                const int parts = p1 - p0 + 1;
                constexpr int BATCH = 8;      // parts loaded together: few would wait for the memory, one after another
                for (int d = 4 * threadIdx.x; d < heads * HD; d += 4 * AT_THREADS) {
                    const int h = d / HD;
                    float top = -INFINITY, den = 0.0f;
                    bool bad = false;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int k0 = 0; k0 < parts; k0 += BATCH) {
                        float2 ml[BATCH];
                        float4 v[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; ++i) {
                            const int k = k0 + i;
                            const float *p = part + (size_t)(k ? 2 * k - 1 : 0) * G::SLOT;
                            ml[i] = make_float2(0.0f, 0.0f);
                            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (k < parts) {
                                ml[i] = __ldcg(reinterpret_cast<const float2 *>(p) + h);
                                v[i] = __ldcg(reinterpret_cast<const float4 *>(p + 2 * KV4_HEADS + d));
                            }
                        }
                        float to = top;
#pragma unroll
                        for (int i = 0; i < BATCH; ++i) {
                            if (ml[i].y != 0.0f) to = fmaxf(to, ml[i].x);
                            bad |= ml[i].y < 0.0f;
                        }
                        const float fix = den != 0.0f ? at_ex2(top - to) : 0.0f;
                        top = to;
                        den *= fix;
                        sum.x *= fix, sum.y *= fix, sum.z *= fix, sum.w *= fix;
#pragma unroll
                        for (int i = 0; i < BATCH; ++i) {
                            const float f = at_ex2(ml[i].x - top);
                            if (ml[i].y != 0.0f) {
                                den = fmaf(ml[i].y, f, den);
                                sum.x = fmaf(v[i].x, f, sum.x), sum.y = fmaf(v[i].y, f, sum.y);
                                sum.z = fmaf(v[i].z, f, sum.z), sum.w = fmaf(v[i].w, f, sum.w);
                            }
                        }
                    }
                    if (bad) at_store4<T>(out + d, a.wide, 0.0f, 0.0f, 0.0f, 0.0f);
                    else at_store4<T>(out + d, a.wide, sum.x / den, sum.y / den, sum.z / den, sum.w / den);
                }
            }
        }
        __syncthreads();                      // the join's memory is free again
        if (lane == 0) w = after;
        __syncwarp();
    }
    zeros();
    if (!ok)                                  // copies in flight land before the CTA leaves
        for (; ahead > 0; --ahead) {
            mbar_wait_bounded(&full[warp][slot], phase, c.status, HOLO_E_TIMEOUT);
            if (++slot == STAGES) slot = 0, phase ^= 1;
        }
}

template <typename T, int HD>
bool launch(const Kv4View &view, AtArgs a, int sms, cudaStream_t st) {
    using G = AtGeom<HD>;
    static bool configured[16] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 16 || !configured[dev]) {
        if (cudaFuncSetAttribute(kv4_attn_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM) != cudaSuccess)
            return false;
        if (dev < 16) configured[dev] = true;
    }
    // no more CTAs than the sequences could keep busy if their tables were full
    const long long items = (long long)a.n * view.n_kv * a.chunks;
    const long long most = ((long long)view.max_pages * view.page_tokens + AT_UNIT_POS * AT_MIN - 1) / (AT_UNIT_POS * AT_MIN);
    const int grid = (int)min((long long)min(sms * G::CTAS, KV4_MAX_CTAS), items * most);
    return holo_launch_early(kv4_attn_kernel<T, HD>, grid, AT_THREADS, G::SMEM, st, view, a) == cudaSuccess;
}

template <typename T>
bool launch_hd(const holo_kv4 *c, const Kv4View &view, const AtArgs &a, int sms, cudaStream_t st) {
    switch (c->head_dim) {
    case 64: return launch<T, 64>(view, a, sms, st);
    case 128: return launch<T, 128>(view, a, sms, st);
    default: return launch<T, 256>(view, a, sms, st);
    }
}

}  // namespace

extern "C" int cuda_kv4_attention(const holo_kv4 *c, int layer, void *out, const void *q, int type, long long q_row,
                                  long long out_row, int n_heads, float scale, const int *seqs, int n) {
    const char *what = "cuda_kv4_attention";
    Kv4View view;
    Kv4Work work;
    cudaStream_t st;
    if (!kv4_begin(c, layer, what, view, st, &work)) return cuda_last_status();
    auto refuse = [&](int code) {
        holo_set_status(code, what);
        return code;
    };
    if (type != HOLO_DT_F32 && type != HOLO_DT_F16 && type != HOLO_DT_BF16) return refuse(HOLO_E_UNSUPPORTED);
    const long long dense = (long long)n_heads * c->head_dim;
    if (q_row == 0) q_row = dense;
    if (out_row == 0) out_row = dense;
    const int size = type == HOLO_DT_F32 ? 4 : 2;
    if (n_heads <= 0 || n_heads % c->n_kv_heads || n < 0 || n > c->max_seqs || q_row < dense || out_row < dense ||
        !(scale >= 0.0f) || (n > 0 && (!out || !q)) || ((uintptr_t)q | (uintptr_t)out) % size)
        return refuse(HOLO_E_ARG);
    const int group = n_heads / c->n_kv_heads;
    if (group > KV4_MAX_GROUP) return refuse(HOLO_E_UNSUPPORTED);
    if (n == 0) return HOLO_OK;
    AtArgs a;
    a.out = out, a.q = q, a.q_row = q_row, a.out_row = out_row, a.seqs = seqs;
    a.n = n, a.n_heads = n_heads, a.group = group, a.chunks = (group + KV4_HEADS - 1) / KV4_HEADS;
    a.scale = scale == 0.0f ? 1.0f / sqrtf((float)c->head_dim) : scale;
    // places of the list, at most: counted in an int
    const long long units = ((long long)c->max_pages * c->page_tokens + AT_UNIT_POS - 1) / AT_UNIT_POS + AT_ITEM;
    if (units * n * c->n_kv_heads * a.chunks > 0x40000000LL) return refuse(HOLO_E_UNSUPPORTED);
    a.page_magic = view.page_blocks == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + view.page_blocks - 1) / view.page_blocks);
    a.wide = (uintptr_t)out % 16 == 0 && out_row * size % 16 == 0;
    a.q_wide = (uintptr_t)q % 16 == 0 && q_row * size % 16 == 0;
    a.counters = work.counters, a.partial = work.partial;
    // Where there may be fewer items than CTAs, each CTA has one at most and its cost is the same for all.  (Two CTAs an SM, as at
    // 128 dims; the three at 64 and the one at 256 have not been measured apart.)
    a.item_cost = (long long)n * c->n_kv_heads * a.chunks >= holo_dev()->sms * 2 ? AT_ITEM : 0;
    const int sms = holo_dev()->sms;
    bool done;
    switch (type) {
    case HOLO_DT_F32: done = launch_hd<float>(c, view, a, sms, st); break;
    case HOLO_DT_F16: done = launch_hd<__half>(c, view, a, sms, st); break;
    default: done = launch_hd<__nv_bfloat16>(c, view, a, sms, st); break;
    }
    if (!done) {
        holo_check_launch(what);
        return cuda_last_status();
    }
    return kv4_end(what);
}
