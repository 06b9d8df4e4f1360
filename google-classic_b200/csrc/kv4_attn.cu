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
//   values   Codes of two positions become fp16 (n - 8) with one or and one
//            subtraction a pair (exact); A: 16 dims, B: the softmax weights of
//            8 heads times the position's scale of the group, transposed by
//            movmatrix.
// Only the weights are rounded (to fp16; for fp32 rows a second fp16 term
// carries the rest, as for q).  So that they use fp16's range whatever the
// values' size, they are scaled by a power of two that follows the largest
// scale seen; a head's q is scaled by the power of two of its largest value.
//
// The units of work, 32 positions of 8 heads of one KV head, of all sequences form one
// list that is cut evenly over the CTAs (ragged batches stay balanced).  Each warp
// streams every fourth unit of its CTA's part through a ring of its own, one
// bulk copy a block of 16 positions, its table entry loaded a unit ahead, and
// keeps a running maximum, sum and output; warps join in shared memory.  A
// list item that is cut leaves partial results, and the CTA that comes last joins them in
// their order, so the result does not depend on timing.
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int AT_WARPS = 4, AT_THREADS = 32 * AT_WARPS;
constexpr int AT_UNIT = 2;                     // blocks of 16 positions a unit
constexpr int AT_UNIT_POS = AT_UNIT * KV4_BLOCK;
constexpr int AT_WHOLE = 16;                   // items of up to so many units are not cut
constexpr float AT_SHIFT = 256.0f;             // weights times scales lie below this

template <int HD> struct AtGeom {
    static constexpr int NB = HD / KV4_GROUP;
    static constexpr int BLOCK_BYTES = kv4_block_bytes(HD);
    static constexpr int STAGES = HD == 64 ? 4 : 3;
    static constexpr int RING = AT_WARPS * STAGES * AT_UNIT * BLOCK_BYTES;
    static constexpr int JOIN = AT_WARPS * KV4_HEADS * HD * 4;
    static constexpr int SMEM = RING + JOIN;
    static constexpr int CTAS = HD == 256 ? 1 : 3;   // an SM
    static constexpr int SLOT = KV4_HEADS * (HD + 2);   // floats of a partial result: m and l of the heads, then the outputs
};

struct AtArgs {
    void *out;
    const void *q;
    long long q_row, out_row;
    const int *seqs;
    int n, n_heads, group, chunks;             // chunks of KV4_HEADS query heads a KV head
    float scale;
    uint64_t page_magic;                       // ceil(2^32 / page_blocks)
    int *counters;
    float *partial;
};

__device__ __forceinline__ float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void at_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t at_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t at_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 at_unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
// two codes, 0..15 each in a half at bit 0 or 4 (mask), as fp16 code - 8 or 16 (code - 8)
template <uint32_t MASK, uint32_t BIAS>
__device__ __forceinline__ uint32_t at_signed(uint32_t x) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "n"(MASK), "n"(0x64006400u));   // (x & MASK) | 1024.0
    const uint32_t bias = BIAS;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&y), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&r);
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

// The list of units: of every sequence, every (KV head, chunk of heads), its
// units.  A walk through the CTA's part, item by item.
struct Walk {
    int i, s, len, units;      // sequence: its place in the list, number, positions, units an item
    int item;                  // KV head * chunks + chunk
    int first, take;           // units of the item in the part
    long long rest;            // units of the part from `first` on
};

__device__ __forceinline__ int at_units(const Kv4View &c, const AtArgs &a, int i, int &s, int &len) {
    s = a.seqs ? __ldg(a.seqs + i) : i;
    len = 0;
    if (s < 0 || s >= c.max_seqs) {
        s = -1;
        return 0;
    }
    len = max(0, min(__ldg(c.lens + s), c.max_pages * c.page_tokens));
    return (len + AT_UNIT_POS - 1) / AT_UNIT_POS;
}
__device__ __forceinline__ void at_clip(Walk &w) { w.take = (int)min((long long)(w.units - w.first), w.rest); }
// the next item of the part; rest 0 at its end
__device__ __forceinline__ void at_next(const Kv4View &c, const AtArgs &a, Walk &w) {
    w.rest -= w.take;
    w.first = w.take = 0;
    if (w.rest <= 0) return;
    if (++w.item == c.n_kv * a.chunks) {
        w.item = 0;
        do {
            if (++w.i >= a.n) {
                w.rest = 0;
                return;
            }
            w.units = at_units(c, a, w.i, w.s, w.len);
        } while (w.units == 0);
    }
    at_clip(w);
}

// inclusive sum over the CTA
__device__ __forceinline__ long long at_scan(long long v, long long *sh, long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    total = 0;
    for (int w = 0; w < AT_WARPS; ++w) {
        if (w < warp) v += sh[w];
        total += sh[w];
    }
    return v;
}

template <typename T, int HD>
__global__ void __launch_bounds__(AT_THREADS, AtGeom<HD>::CTAS)
kv4_attn_kernel(const __grid_constant__ Kv4View c, const __grid_constant__ AtArgs a) {
    using G = AtGeom<HD>;
    constexpr int NB = G::NB, STAGES = G::STAGES;
    constexpr bool FINE = sizeof(T) == 4;      // fp32 rows: second terms of q and of the weights
    constexpr int TERMS = FINE ? 2 : 1;
    extern __shared__ __align__(128) uint8_t at_smem[];
    __shared__ uint64_t full[AT_WARPS][STAGES];
    __shared__ long long scan[AT_WARPS];
    __shared__ Walk begin;
    __shared__ long long part_start, part_end;
    __shared__ float join_m[AT_WARPS][KV4_HEADS], join_l[AT_WARPS][KV4_HEADS];
    __shared__ int last;
    float *join = reinterpret_cast<float *>(at_smem + G::RING);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t *ring = at_smem + (size_t)warp * STAGES * AT_UNIT * G::BLOCK_BYTES;

    if (lane < STAGES) mbar_init(&full[warp][lane], 1);
    fence_barrier_init();

    // ---- the CTA's part of the list ----
    const int items = c.n_kv * a.chunks;
    long long all = 0;
    for (int i0 = 0; i0 < a.n; i0 += AT_THREADS) {
        const int i = i0 + threadIdx.x;
        int s, len, u = 0;
        if (i < a.n) {
            u = at_units(c, a, i, s, len);
            if (s < 0 && blockIdx.x == 0) kv4_report(c.status, HOLO_E_ARG);
        }
        long long total;
        at_scan((long long)u * items, scan, total);
        all += total;
    }
    // no more CTAs than leave each warp a unit
    const int ctas = (int)min((long long)gridDim.x, max(1LL, (all + AT_WARPS - 1) / AT_WARPS));
    // sequences without positions: zeros (a sequence number out of range: left alone)
    for (int i = blockIdx.x; i < a.n; i += gridDim.x) {
        int s, len;
        if (at_units(c, a, i, s, len) == 0 && s >= 0)
            for (int d = threadIdx.x; d < a.n_heads * HD; d += AT_THREADS)
                ((T *)a.out)[i * a.out_row + d] = kv4_from_float<T>(0.0f);
    }
    if ((int)blockIdx.x >= ctas) return;
    // Its part [u0, u1): the even cuts of the list, moved down to the item's start
    // where the item is short.  Cuts inside longer items stay, so that the parts that an item spans follow from them.
    const long long cut0 = all * blockIdx.x / ctas, cut1 = all * (blockIdx.x + 1) / ctas;
    if (threadIdx.x == 0) part_end = all;
    {
        long long before = 0;
        for (int i0 = 0; i0 < a.n && before <= cut1; i0 += AT_THREADS) {
            const int i = i0 + threadIdx.x;
            int s = -1, len = 0, u = 0;
            if (i < a.n) u = at_units(c, a, i, s, len);
            long long total;
            const long long end = before + at_scan((long long)u * items, scan, total), start = end - (long long)u * items;
            if (start <= cut0 && cut0 < end) {
                Walk w;
                w.i = i, w.s = s, w.len = len, w.units = u;
                w.item = (int)((cut0 - start) / u);
                w.first = u > AT_WHOLE ? (int)((cut0 - start) % u) : 0;
                begin = w;
                part_start = start + (long long)w.item * u + w.first;
            }
            if (start <= cut1 && cut1 < end) part_end = u > AT_WHOLE ? cut1 : start + (cut1 - start) / u * u;
            before += total;
        }
        __syncthreads();
    }
    const long long u0 = part_start, u1 = part_end;
    if (u0 >= u1) return;
    Walk head = begin;
    head.rest = u1 - u0;
    at_clip(head);

    // ---- the warp's loads: unit `unit` of item `load` ----
    Walk load = head;
    int unit = load.first + warp;
    auto settle = [&]() {                     // to the next unit that there is
        while (load.rest > 0 && unit >= load.first + load.take) {
            at_next(c, a, load);
            unit = load.first + warp;
        }
    };
    settle();
    int entry = -1;                           // lanes 0 and 1: the page of their block of it
    int block = 0;                            // and the block in the sequence
    auto look_up = [&]() {
        block = unit * AT_UNIT + lane;
        if (load.rest > 0 && lane < AT_UNIT && block * KV4_BLOCK < load.len)
            entry = __ldg(c.tables + (size_t)load.s * c.max_pages + (int)((block * a.page_magic) >> 32));
    };
    look_up();
    int issued = 0;
    auto issue = [&]() {                      // its copies, and the table entries of the next one
        if (load.rest <= 0) return;
        const int slot = issued % STAGES;
        const int blocks = min(AT_UNIT, (load.len - unit * AT_UNIT_POS + KV4_BLOCK - 1) / KV4_BLOCK);
        if (lane == 0) mbar_arrive_expect_tx(&full[warp][slot], blocks * G::BLOCK_BYTES);
        __syncwarp();
        if (lane < blocks) {
            if (entry < 0 || entry >= c.n_pages) {
                kv4_report(c.status, HOLO_E_ARG);
                entry = 0;
            }
            const int in_page = block - (int)((block * a.page_magic) >> 32) * c.page_blocks;
            const uint8_t *src = kv4_block(c, HD, entry, load.item / a.chunks, in_page);
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                :: "r"(smem_addr(ring + (slot * AT_UNIT + lane) * G::BLOCK_BYTES)), "l"(src), "r"(G::BLOCK_BYTES),
                   "r"(smem_addr(&full[warp][slot])) : "memory");
        }
        ++issued;
        unit += AT_WARPS;
        settle();
        look_up();
    };
    __syncwarp();
    for (int k = 0; k < STAGES; ++k) issue();

    // ---- items ----
    int used = 0;
    bool ok = true;
    for (Walk w = head; w.rest > 0; at_next(c, a, w)) {
        const int kvh = w.item / a.chunks, head0 = kvh * a.group + (w.item % a.chunks) * KV4_HEADS;
        const int heads = min(KV4_HEADS, (kvh + 1) * a.group - head0);
        // q of head g: quarter t of every group, times a power of two; B fragments of the two steps of a group
        uint32_t qf[TERMS][NB][2][2];
        float start[NB][2], factor[2];        // of heads 2 t and 2 t + 1
        {
            float qv[NB][8], top = 0.0f;
            const T *q = (const T *)a.q + w.i * a.q_row + (long long)(head0 + g) * HD + 8 * t;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    qv[b][e] = g < heads ? kv4_to_float<T>(q[32 * b + e]) : 0.0f;
                    top = fmaxf(top, fabsf(qv[b][e]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(11 - exponent) brings the largest to [2^11, 2^12)
            const int e0 = max(12, (int)(__float_as_uint(top) >> 23));
            const float up = __uint_as_float((uint32_t)(265 - e0) << 23);
            const float down = __uint_as_float((uint32_t)(e0 - 11) << 23) * a.scale * 1.4426950408889634f * 16777216.0f;
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

        for (int u = w.first + warp; u < w.first + w.take; u += AT_WARPS) {
            const int slot = used % STAGES;
            ok = ok && mbar_wait_bounded(&full[warp][slot], used / STAGES & 1, c.status, HOLO_E_TIMEOUT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++used;
            const uint8_t *buf = ring + slot * AT_UNIT * G::BLOCK_BYTES;
            const int left = w.len - u * AT_UNIT_POS;   // positions of the sequence from the unit's first on
            // scores of positions g, g + 8 (+ 16 a block), heads 2 t and 2 t + 1
            float s[AT_UNIT][4];
            AtWords<NB / 2> dv[AT_UNIT][2];
            uint32_t dmax = 0;
#pragma unroll
            for (int k = 0; k < AT_UNIT; ++k) {
                const uint8_t *blk = buf + k * G::BLOCK_BYTES;
                const bool live[2] = {16 * k + g < left, 16 * k + g + 8 < left};
                const AtWords<NB> w0 = at_lds<NB>(blk + g * (HD / 2) + t * 4 * NB);
                const AtWords<NB> w1 = at_lds<NB>(blk + (g + 8) * (HD / 2) + t * 4 * NB);
                const AtWords<NB / 2> d0 = at_lds<NB / 2>(blk + kv4_off_dk(HD) + g * 2 * NB);
                const AtWords<NB / 2> d1 = at_lds<NB / 2>(blk + kv4_off_dk(HD) + (g + 8) * 2 * NB);
                dv[k][0] = at_lds<NB / 2>(blk + kv4_off_dv(HD) + g * 2 * NB);
                dv[k][1] = at_lds<NB / 2>(blk + kv4_off_dv(HD) + (g + 8) * 2 * NB);
                float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float acc[4] = {start[b][0], start[b][1], start[b][0], start[b][1]};
                    const uint32_t x = w0.w[b], y = w1.w[b], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
                    for (int f = 0; f < TERMS; ++f) {
                        at_mma(acc, x & 0x000f000fu, y & 0x000f000fu, x8 & 0x000f000fu, y8 & 0x000f000fu, qf[f][b][0][0],
                               qf[f][b][0][1]);
                        at_mma(acc, x & 0x00f000f0u, y & 0x00f000f0u, x8 & 0x00f000f0u, y8 & 0x00f000f0u, qf[f][b][1][0],
                               qf[f][b][1][1]);
                    }
                    const float2 e0 = at_unpack(d0.w[b >> 1]), e1 = at_unpack(d1.w[b >> 1]);
                    const float s0 = b & 1 ? e0.y : e0.x, s1 = b & 1 ? e1.y : e1.x;
                    r[0] = fmaf(s0, acc[0], r[0]);
                    r[1] = fmaf(s0, acc[1], r[1]);
                    r[2] = fmaf(s1, acc[2], r[2]);
                    r[3] = fmaf(s1, acc[3], r[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[k][e] = live[e >> 1] ? r[e] * factor[e & 1] : -INFINITY;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i) {
                        if (!live[x]) dv[k][x].w[i] = 0;   // whatever lies there
                        dmax = __vmaxu2(dmax, dv[k][x].w[i] & 0x7fff7fffu);
                    }
            }
            // maxima of the unit, over positions (and of the scales, over all)
            float mn[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mn[x] = fmaxf(fmaxf(s[0][x], s[0][x + 2]), fmaxf(s[1][x], s[1][x + 2]));
#pragma unroll
                for (int i = 4; i < 32; i <<= 1) mn[x] = fmaxf(mn[x], __shfl_xor_sync(0xffffffffu, mn[x], i));
                mn[x] = fmaxf(mn[x], m[x]);
            }
            const uint32_t big = __reduce_max_sync(0xffffffffu, max(dmax & 0xffffu, dmax >> 16));
            const int pn = max(power, (int)(big >> 10) - 14);   // fp16 exponent field e: below 2^(e - 14)
            if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1]) || pn > power) {
                const float lower = __uint_as_float((uint32_t)(127 + power - pn) << 23);   // 2^(power - pn)
                float fix[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    fix[x] = mn[x] > m[x] ? at_ex2(m[x] - mn[x]) : 1.0f;
                    l[x] *= fix[x];
                    fix[x] *= lower;
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
            const float unit_scale = __uint_as_float((uint32_t)(127 - power) << 23) * AT_SHIFT;
            float sub[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) sub[x] = m[x] == -INFINITY ? 0.0f : m[x];
#pragma unroll
            for (int k = 0; k < AT_UNIT; ++k) {
                const uint8_t *blk = buf + k * G::BLOCK_BYTES;
                if (16 * k >= left) break;    // a block that was not loaded
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = at_ex2(s[k][e] - sub[e & 1]);
                    l[e & 1] += p[e];
                }
                // codes of positions 2 t, 2 t + 1 and 2 t + 8, 2 t + 9, values 4 g .. 4 g + 3 of every group
                const uint8_t *v = blk + kv4_off_v(HD) + ((g >> 1) * 8 * 2 + (g & 1)) * 4 * NB;
                const AtWords<NB> v0 = at_lds<NB>(v + t * 8 * NB), v1 = at_lds<NB>(v + (t + 4) * 8 * NB);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float2 e0 = at_unpack(dv[k][0].w[b >> 1]), e1 = at_unpack(dv[k][1].w[b >> 1]);
                    const float s0 = (b & 1 ? e0.y : e0.x) * unit_scale, s1 = (b & 1 ? e1.y : e1.x) * unit_scale;
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
                    constexpr uint32_t LOW = 0x5410, HIGH = 0x7632;
                    const uint32_t pick = b & 1 ? HIGH : LOW;
                    const uint32_t x0 = __byte_perm(v0.w[b >> 1], v0.w[NB / 2 + (b >> 1)], pick);
                    const uint32_t x1 = __byte_perm(v1.w[b >> 1], v1.w[NB / 2 + (b >> 1)], pick);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t z0 = x0 >> (8 * x), z1 = x1 >> (8 * x);
                        const uint32_t a0 = at_signed<0x000f000fu, 0x64086408u>(z0), a1 = at_signed<0x00f000f0u, 0x64806480u>(z0);
                        const uint32_t a2 = at_signed<0x000f000fu, 0x64086408u>(z1), a3 = at_signed<0x00f000f0u, 0x64806480u>(z1);
#pragma unroll
                        for (int f = 0; f < TERMS; ++f) at_mma(o[b][x], a0, a1, a2, a3, pf[f][0], pf[f][1]);
                    }
                }
            }
            __syncwarp();                     // the slot has been read
            issue();
        }

        // ---- join the warps ----
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], i);
        if (g == 0) {
            join_m[warp][2 * t] = m[0], join_m[warp][2 * t + 1] = m[1];
            join_l[warp][2 * t] = l[0], join_l[warp][2 * t + 1] = l[1];
        }
        const float back = __uint_as_float((uint32_t)(127 + power) << 23) / AT_SHIFT;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)   // values 32 b + 4 g + 2 x (and + 1, 16 times as large), heads 2 t + (e & 1)
                    join[(warp * KV4_HEADS + 2 * t + (e & 1)) * HD + 32 * b + 4 * g + 2 * x + (e >> 1)] =
                        o[b][x][e] * (e & 2 ? back * 0.0625f : back);
        __syncthreads();
        const bool whole = w.first == 0 && w.take == w.units;
        const int slot0 = w.first > 0 ? 0 : 1;
        float *mine = a.partial + ((size_t)blockIdx.x * 2 + slot0) * G::SLOT;
        for (int d = threadIdx.x; d < heads * HD; d += AT_THREADS) {
            const int h = d / HD;
            float top = -INFINITY, sum = 0.0f, den = 0.0f;
#pragma unroll
            for (int i = 0; i < AT_WARPS; ++i)
                if (join_l[i][h] != 0.0f) top = fmaxf(top, join_m[i][h]);
#pragma unroll
            for (int i = 0; i < AT_WARPS; ++i)
                if (join_l[i][h] != 0.0f) {
                    const float f = at_ex2(join_m[i][h] - top);
                    sum = fmaf(join[(i * KV4_HEADS + h) * HD + d % HD], f, sum);
                    den = fmaf(join_l[i][h], f, den);
                }
            if (whole) {
                ((T *)a.out)[w.i * a.out_row + (long long)(head0 + h) * HD + d % HD] = kv4_from_float<T>(sum / den);
            } else {
                mine[2 * KV4_HEADS + d] = sum;
                if (d % HD == 0) mine[2 * h] = top, mine[2 * h + 1] = den;
            }
        }
        if (!whole) {
            // the item's units lie in the parts of CTAs c0 .. c1: part k holds unit u where k = ((u + 1) * ctas - 1) / all
            const long long begins = (w.first > 0 ? u0 - w.first : u1 - w.rest);
            const int c0 = (int)(((begins + 1) * ctas - 1) / all), c1 = (int)(((begins + w.units) * ctas - 1) / all);
            int *counter = a.counters + (size_t)w.i * items + w.item;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last = atomicAdd(counter, 1) == c1 - c0;
            __syncthreads();
            if (last) {
                __threadfence();
                if (threadIdx.x == 0) *counter = 0;
                for (int d = threadIdx.x; d < heads * HD; d += AT_THREADS) {
                    const int h = d / HD;
                    float top = -INFINITY, sum = 0.0f, den = 0.0f;
                    for (int k = c0; k <= c1; ++k) {
                        const float *p = a.partial + ((size_t)k * 2 + (k == c0 ? 1 : 0)) * G::SLOT;
                        const float pm = __ldcg(p + 2 * h), pl = __ldcg(p + 2 * h + 1), po = __ldcg(p + 2 * KV4_HEADS + d);
                        if (pl != 0.0f) {
                            const float mx = fmaxf(top, pm), f = at_ex2(pm - mx), fo = sum == 0.0f && den == 0.0f ? 0.0f : at_ex2(top - mx);
                            sum = fmaf(po, f, sum * fo);
                            den = fmaf(pl, f, den * fo);
                            top = mx;
                        }
                    }
                    ((T *)a.out)[w.i * a.out_row + (long long)(head0 + h) * HD + d % HD] = kv4_from_float<T>(sum / den);
                }
            }
        }
        __syncthreads();                      // the join's memory is free again
    }
    if (!ok)                                  // copies in flight land before the CTA leaves
        for (int k = used; k < issued; ++k)
            mbar_wait_bounded(&full[warp][k % STAGES], k / STAGES & 1, c.status, HOLO_E_TIMEOUT);
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
    const int grid = min(sms * G::CTAS, KV4_MAX_CTAS);
    kv4_attn_kernel<T, HD><<<grid, AT_THREADS, G::SMEM, st>>>(view, a);
    return true;
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
    a.page_magic = (((uint64_t)1 << 32) + view.page_blocks - 1) / view.page_blocks;
    a.counters = work.counters, a.partial = work.partial;
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
