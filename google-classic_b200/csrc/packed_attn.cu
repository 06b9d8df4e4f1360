// packed_attn.cu -- causal attention of whole prompts of different lengths
// that lie one after another in the rows (holo_b200.h, cuda_attention_packed).
//
// Two kernels.  The tensor-core kernel takes rows that TMA can address (bases
// and strides of whole 16 bytes); other rows take one warp a row and head, which is
// about a hundredth as fast (four sequences of 1024, 16 heads of 128 over 8, bf16:
// 29.5 us and 2.9 ms) but reads any row in place.
//
// Tensor-core kernel: persistent CTAs, one an SM; an item of work is 256 query
// rows of one head and sequence, as two tiles of 128, which walk the sequence's
// keys in steps of 64 up to the diagonal.  (Head size 256: one tile, whose O takes
// the room of two, and a ring of 64-key tiles.)
//   S_t = Q_t K^T    tcgen05.mma, Q_t and K from shared memory, S_t in TMEM
//   P_t = 2^(c S_t - m)   a thread a row: it reads its row of S_t, keeps the
//                    row's maximum m and sum l, and writes P_t (16 bits) over S_t
//   O_t += P_t V     tcgen05.mma, P_t from TMEM, V from shared memory as it
//                    lies (keys by dims: the transposed operand), O_t in TMEM
// TMEM holds O_0, O_1 and two S of 64 keys for each tile, so that a step's
// scores are there before the softmax of the step before ends, and neither the
// softmax nor the tensor core waits through the other's latency.  (Steps of 128
// keys leave room for one S a tile: then each tile's chain, softmax 2000 cycles, P V,
// 290 to its end, Q K^T, 350 to its reader, sets the pace, 4100 cycles a pair of
// tiles; their MMAs are 2048.  At N = 64 Q K^T is bound by shared memory, 48 cycles
// an MMA and not 32: 2560 cycles.)
// Warps 0-3 and 4-7 are the softmax of tile 0 and 1 (TMEM lane = query row),
// warps 8 and 9 issue the MMAs of tile 0 and 1, warp 10 the TMA loads of Q and of
// K and V into a ring of tiles of 128 keys, warp 11 finds the items and checks V
// (below).  All of them run on into the next item: its loads and first scores
// are under way while the softmax warps write the rows of the last.
// One sequence of 16383 (64 heads of 128 over 8, bf16) runs at 1080 TFLOP/s and the
// board's power (SM clock 1.6 GHz at 1000 W), 16384 at head size 256 (16 heads over 2) at
// 1104, eight of up to 4096 at 895.  What bounds the last, and all at full clock (zeros in every
// row), is the two tiles' chains: a step takes 1645 cycles, 1270 of them the softmax's own, where
// the MMAs of a pair need 1280, so the tensor pipe is busy for half of them; and an item's
// ends, where only one of softmax and tensor core has work: 5000 to 5800 cycles, 30,000 of a CTA's
// 150,000 with sequences of up to 2048.  Four of 1024 (16 heads over 8): 29.5 us, 580.
// O_t is rescaled only when a row's maximum has grown by more than 2^8 since
// the last time, which after the first key tiles is rare.  In bf16 P's rounding is
// relative whatever its size.  In fp16 P is taken times 2^7, up to 2^15 then, so that weights
// down to 2^-32 of the largest count (2^-25 without, and 100,000 such are 0.3 % of a row).
//
// A masked place never counts.  Its P is an exact 0, which an infinite or NaN
// value of V would still make NaN: where a row's result is not finite, the CTA
// goes through its items a second time with care.  Then warp 11 sets the values
// of V that are not finite to 0 before the tensor core reads a tile, and keeps, for each
// dim, the first key with a NaN, an infinity and a negative one; the rows from that key
// on have that as their result (a weight is never 0 in the formula).
// A NaN score needs none of this: it makes its row NaN by itself.  Where the
// cleaned sums still overflow fp32 (bf16 values near the largest, times weights before the
// division), a third pass takes V by 2^-32 and the sums by 2^32.
// A sequence of 4096 (2 heads over 1 of 128, f16): 60 to 67 us, 270 with two such values, 1,700 with all of V
// NaN; of 16,383 (64 heads over 8, bf16): 3.5, 15.7 and 101 ms.
#include "holo_common.cuh"
#include "mv_unit.cuh"
#include "tc_util.cuh"

#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>
#include <type_traits>

namespace {

using namespace holo_tc;

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(float x, __half &y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }

struct PackedArgs {
    void *out;
    const void *q, *k, *v;
    const int *cu;
    float *lse;
    int n_seqs, total, n_heads, group;
    float scale;
    long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    int item_rows;                     // 256, or 128: one tile an item, where that many items are wanted
    int *status;
};

// first row and length of sequence s, inside the rows whatever cu says
__device__ __forceinline__ void packed_seq(const PackedArgs &a, int s, int &first, int &len) {
    first = max(0, __ldcg(a.cu + s));
    len = max(0, min(a.total, __ldcg(a.cu + s + 1)) - first);
}

// ---------------------------------------------------------------------------
// one warp a row and head: lane l holds dims l, l + 32, ...; online softmax
// over the row's own keys; where its sums are not finite, once more with the values that are not apart
// ---------------------------------------------------------------------------
template <typename T, int HD>
__global__ void __launch_bounds__(128)
packed_simple_kernel(const __grid_constant__ PackedArgs a) {
    constexpr int NB = HD / 32;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, lane = threadIdx.x & 31;
    if (row >= a.total) return;
    int lo = 0, hi = a.n_seqs;   // the last s with cu[s] <= row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(a.cu + mid) <= row) lo = mid;
        else hi = mid;
    }
    int first, len;
    packed_seq(a, lo, first, len);
    if (row < first || row >= first + len) return;
    const T *q = (const T *)a.q + row * a.q_row + h * a.q_head;
    float qv[NB], acc[NB], bad[NB], m, l;
#pragma unroll
    for (int b = 0; b < NB; ++b) qv[b] = to_float(q[32 * b + lane]) * a.scale;
    auto walk = [&](auto apart) {   // apart: values that are not finite into `bad`, without weights
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = bad[b] = 0.0f;
        for (int j = first; j <= row; ++j) {
            const T *k = (const T *)a.k + j * a.k_row + h / a.group * a.k_head;
            const T *v = (const T *)a.v + j * a.v_row + h / a.group * a.v_head;
            float dot = 0.0f, x[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                dot = fmaf(qv[b], to_float(k[32 * b + lane]), dot);
                x[b] = to_float(v[32 * b + lane]);
                if (apart && !isfinite(x[b])) bad[b] += x[b], x[b] = 0.0f;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (dot == -INFINITY) continue;   // weight 0
            const float mn = fmaxf(m, dot), fix = expf(m - mn), e = expf(dot - mn);
            l = l * fix + e;
            m = mn;
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b] = fmaf(e, x[b], acc[b] * fix);
        }
    };
    walk(std::false_type());
    bool finite = true;
#pragma unroll
    for (int b = 0; b < NB; ++b) finite = finite && isfinite(acc[b]);
    if (!__all_sync(0xffffffffu, finite)) walk(std::true_type());
    T *o = (T *)a.out + row * a.out_row + h * a.out_head;
#pragma unroll
    for (int b = 0; b < NB; ++b) from_float(acc[b] / l + bad[b], o[32 * b + lane]);
    if (a.lse && lane == 0) a.lse[(size_t)h * a.total + row] = m + logf(l);
}

template <typename T>
void launch_simple(const PackedArgs &a, int hd, cudaStream_t st) {
    const dim3 grid((a.total + 3) / 4, a.n_heads);
    switch (hd) {
    case 64: packed_simple_kernel<T, 64><<<grid, 128, 0, st>>>(a); break;
    case 128: packed_simple_kernel<T, 128><<<grid, 128, 0, st>>>(a); break;
    default: packed_simple_kernel<T, 256><<<grid, 128, 0, st>>>(a); break;
    }
}

// ---------------------------------------------------------------------------
// tensor-core kernel
// ---------------------------------------------------------------------------
constexpr int PK_ROWS = 128;           // query rows a tile (MMA M)
constexpr int PK_STEP = 64;            // keys a step (MMA N of S, K of P V)
constexpr int PK_THREADS = 384;        // three warpgroups
// registers a thread, of 384 * 168 at launch: 2 * 208 + 88 = 3 * 168
constexpr int PK_SOFTMAX_REGS = 208, PK_OTHER_REGS = 88;
static_assert(2 * PK_SOFTMAX_REGS + PK_OTHER_REGS <= 3 * 168, "a split above the launch's registers would wait for ever");
constexpr uint32_t PK_TMEM_COLS = 512; // two S_0, two S_1 (64 columns each), O_0, O_1 (128; O_0 256): all, so they begin at 0
constexpr float PK_GROWTH = 8.0f;      // log2 of what a row's maximum may grow by before its O is rescaled
constexpr int PK_STAGES = 5;           // ring of K and V tiles
constexpr float PK_DOWN = 1.0f / 4294967296.0f;   // 2^-32: of V in the third pass

template <int HD> struct PkGeom {
    static constexpr int TILES = HD == 256 ? 1 : 2;   // query tiles an item: a second O of 256 columns has no room
    static constexpr int KEYS = HD == 256 ? 64 : 128; // keys a tile of the ring
    static constexpr int STEPS = KEYS / PK_STEP;      // steps a tile of the ring
    static constexpr int Q_TILE = PK_ROWS * HD * 2, KV_TILE = KEYS * HD * 2;   // bytes
    static constexpr size_t SMEM = 1024 + (size_t)TILES * Q_TILE + (size_t)PK_STAGES * KV_TILE;
};

// Load i of an item of n ring tiles of K and of V: which side, and its tile j.
// Tiles of two steps come as K_0, V_0, K_1, V_1, ...; of one step as K_0, K_1,
// V_0, K_2, V_1, ..., since scores are taken two steps ahead.
template <int STEPS> __device__ __forceinline__ bool pk_is_value(int i, int n, int &j) {
    if (STEPS == 2) {
        j = i >> 1;
        return i & 1;
    }
    const bool v = i == 2 * n - 1 || (i >= 2 && (i & 1) == 0);
    j = i == 2 * n - 1 ? n - 1 : v ? i / 2 - 1 : i < 2 ? i : (i + 1) / 2;
    return v;
}

struct PkWork {
    int first, len, row0, head;        // the sequence's first row and length; the item's first row in it; len 0: no more
    int careful;                       // 1: V is cleaned; 2: and scaled down
};

struct PkBars {
    uint64_t work_full[2], work_empty[2], q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_done[2][2];
    uint64_t kv_full[PK_STAGES], kv_empty[PK_STAGES], kv_checked[PK_STAGES], bad_known[2], drain[2];
    PkWork work[2];
    int again;                         // the `careful` that a row's result asks for
    uint32_t tmem;
};

__device__ __forceinline__ void pk_tma_load(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar)) : "memory");
}

// Shared-memory descriptors without the address.  K-major (Q and K): as
// sw128_desc.  MN-major, 128-byte-swizzled, of `keys` K rows (V): a K row is 128
// bytes (64 MN values), 8 of them 1024 bytes (SBO), the next 64 MN values `keys`
// rows on (LBO).
constexpr uint64_t PK_DESC_K = ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
constexpr uint64_t pk_desc_mn(int keys) {
    return ((uint64_t)(keys * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ bool pk_elect() {
    uint32_t p;
    asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(p));
    return p != 0;
}

template <typename T> struct PkType;
template <> struct PkType<__half> {
    static constexpr uint32_t AB = 0;   // fp16 operands
    static constexpr float LIFT = 7.0f; // log2 of what P is taken times
    static constexpr uint32_t EXPONENT = 0x7c007c00u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct PkType<__nv_bfloat16> {
    static constexpr uint32_t AB = (1u << 7) | (1u << 10);   // bf16 operands
    static constexpr float LIFT = 0.0f;
    static constexpr uint32_t EXPONENT = 0x7f807f80u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

__device__ __forceinline__ float pk_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 values in one 64-bit register, for the paired fp32 instructions
__device__ __forceinline__ uint64_t pk_pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void pk_split(uint64_t p, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ uint64_t pk_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pk_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// *p = min(*p, v), in shared memory
__device__ __forceinline__ void pk_min16(unsigned short *p, unsigned short v) {
    for (unsigned short old = *(volatile unsigned short *)p; v < old;) {
        const unsigned short got = atomicCAS(p, old, v);
        if (got == old) break;
        old = got;
    }
}

// What is not finite in a row: kinds of values, and row (of the item) from which
// on the item's rows see one; PK_NEVER: none do
enum { PK_NAN, PK_INF, PK_MINUS_INF, PK_KINDS };
constexpr unsigned short PK_NEVER = 0xffff;

// A tile of V in shared memory, its keys from `key0` (of the item's rows) on, as TMA
// has laid it: boxes of 64 dims, rows of 128 bytes, whose 16-byte pieces are exchanged by
// the row's last three bits.  Its values that are not finite become 0 and are
// noted in `seen`; one warp.  scale (bf16): all values by 2^-32.
template <typename T, int HD, int KEYS>
__device__ __forceinline__ void pk_clean_tile(uint8_t *tile, int key0, int len, bool scale,
                                              unsigned short (*seen)[HD]) {
    constexpr uint32_t X = PkType<T>::EXPONENT;
    const int lane = threadIdx.x & 31, piece = lane & 7;
#pragma unroll 1
    for (int box = 0; box < HD / 64; ++box) {
        uint4 *rows = reinterpret_cast<uint4 *>(tile + box * KEYS * 128);
#pragma unroll 4
        for (int r = lane >> 3; r < KEYS; r += 4) {
            uint4 *at = rows + r * 8 + (piece ^ (r & 7));
            const uint4 v = *at;
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            const uint32_t b[4] = {__vcmpeq2(v.x & X, X), __vcmpeq2(v.y & X, X), __vcmpeq2(v.z & X, X), __vcmpeq2(v.w & X, X)};
            const bool any = (b[0] | b[1] | b[2] | b[3]) != 0;
            if (any && key0 + r < len) {
                for (int d = 0; d < 8; ++d) {
                    const uint32_t pair = d < 4 ? (d < 2 ? w[0] : w[1]) : (d < 6 ? w[2] : w[3]);
                    const uint32_t x = d & 1 ? pair >> 16 : pair & 0xffffu;
                    if ((x & X & 0xffffu) != (X & 0xffffu)) continue;
                    const int kind = x & ~X & 0x7fffu ? PK_NAN : x & 0x8000u ? PK_MINUS_INF : PK_INF;
                    pk_min16(&seen[kind][box * 64 + piece * 8 + d], (unsigned short)max(0, key0 + r));
                }
            }
            if (any || scale) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] &= ~b[i];
                    if (std::is_same<T, __nv_bfloat16>::value && scale) {
                        const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]),
                                                         __float2bfloat162_rn(PK_DOWN));
                        w[i] = *reinterpret_cast<const uint32_t *>(&y);
                    }
                }
                *at = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// what row r of an item sees that is not finite becomes its result
template <typename T, int HD>
__device__ __noinline__ void pk_mark_row(T *row, int r, const unsigned short (*seen)[HD]) {
    for (int d = 0; d < HD; ++d) {
        float x = 0.0f;
        if (r >= seen[PK_NAN][d]) x += NAN;
        if (r >= seen[PK_INF][d]) x += INFINITY;
        if (r >= seen[PK_MINUS_INF][d]) x -= INFINITY;
        if (x != 0.0f) from_float(x, row[d]);
    }
}

// Item r of all, heads apart, longest first: the tiles of item_rows rows of all
// sequences in the order of their index, the highest first, and of the
// sequences.  One warp; false if there are no more than r.  `kept`: the lengths of the
// first 256 sequences, eight a lane; `first0`: the first rows of the first 32.
constexpr int PK_KEPT = 8;
__device__ __forceinline__ int pk_len(const PackedArgs &a, int s) {
    int first, len = 0;
    if (s < a.n_seqs) packed_seq(a, s, first, len);
    return len;
}
__device__ __forceinline__ bool pk_find_work(const PackedArgs &a, const int (&kept)[PK_KEPT], int first0, int r, PkWork &w) {
    const int lane = threadIdx.x & 31, shift = a.item_rows == 2 * PK_ROWS ? 8 : 7;
    auto tiles = [&](int len) { return (len + a.item_rows - 1) >> shift; };
    int longest = 0;
#pragma unroll
    for (int i = 0; i < PK_KEPT; ++i) longest = max(longest, kept[i]);
    for (int s = 32 * PK_KEPT + lane; s < a.n_seqs; s += 32) longest = max(longest, pk_len(a, s));
    longest = tiles(__reduce_max_sync(0xffffffffu, longest));
    // tiles of index t or above, over all sequences
    auto from = [&](int t) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PK_KEPT; ++i) n += max(0, tiles(kept[i]) - t);
        for (int s = 32 * PK_KEPT + lane; s < a.n_seqs; s += 32) n += max(0, tiles(pk_len(a, s)) - t);
        return __reduce_add_sync(0xffffffffu, n);
    };
    if (from(0) <= r) return false;
    int lo = 0, hi = longest;   // from(lo) > r >= from(hi)
    int above = 0;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, n = from(mid);
        if (n > r) lo = mid;
        else hi = mid, above = n;
    }
    w.row0 = lo << shift;
    int skip = r - above;       // of the sequences with a tile `lo`
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        int mine = 0;
        if (s0 < 32 * PK_KEPT) {
#pragma unroll
            for (int i = 0; i < PK_KEPT; ++i)
                if (s0 == 32 * i) mine = kept[i];
        } else {
            mine = pk_len(a, s0 + lane);
        }
        const unsigned has = __ballot_sync(0xffffffffu, tiles(mine) > lo);
        const int n = __popc(has);
        if (skip < n) {
            const int src = __fns(has, 0, skip + 1);
            if (s0 == 0) {
                w.first = __shfl_sync(0xffffffffu, first0, src);
                w.len = __shfl_sync(0xffffffffu, mine, src);
            } else {
                packed_seq(a, s0 + src, w.first, w.len);
            }
            return true;
        }
        skip -= n;
    }
    return false;
}

__device__ __forceinline__ float pk_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <typename T, int HD>
__global__ void __launch_bounds__(PK_THREADS, 1)
packed_tc_kernel(const __grid_constant__ PackedArgs a, const __grid_constant__ CUtensorMap qmap,
                 const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using G = PkGeom<HD>;
    extern __shared__ uint8_t pk_smem_raw[];
    __shared__ PkBars B;
    __shared__ unsigned short seen[PK_KINDS][HD];   // of an item with care
    static_assert(sizeof(PkBars) + sizeof(seen) + G::SMEM <= 227 * 1024, "shared memory");
    uint8_t *sq = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pk_smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *skv = sq + G::TILES * G::Q_TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0) {
        tc_alloc(&B.tmem, PK_TMEM_COLS);
    } else if (warp == 1 && lane == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&B.work_full[t], 1);
            mbar_init(&B.work_empty[t], 11);   // warps 8-10 and the softmax's eight
            mbar_init(&B.q_full[t], 1);
            mbar_init(&B.q_empty[t], 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&B.s_full[t][b], 1);
                mbar_init(&B.p_full[t][b], 128);
                mbar_init(&B.o_done[t][b], 1);
            }
            mbar_init(&B.bad_known[t], 1);
            mbar_init(&B.drain[t], 1);
        }
        for (int i = 0; i < PK_STAGES; ++i) {
            mbar_init(&B.kv_full[i], 1);
            mbar_init(&B.kv_empty[i], 3);      // warps 8, 9 and 11 are through with it
            mbar_init(&B.kv_checked[i], 1);
        }
        B.again = 0;
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    early_wait();
    early_next();

    bool ok = true;
    // waits for a phase by its parity: it is the barrier's last but, at most, the one under way
    auto wait = [&](uint64_t *bar, int parity) {
        ok = ok && mbar_wait_bounded(bar, parity & 1, a.status, HOLO_E_TIMEOUT);
        return ok;
    };
    // item k's work, the key tiles of 128 of its two query tiles, and the tiles of the ring
    PkWork w = {};
    int n0 = 0, n1 = 0, n = 0;
    // steps of query tile t: the diagonal key tile's second half is for its rows from 64 on
    auto steps = [&](int t) {
        const int nt = t ? n1 : n0;
        return nt == 0 ? 0 : 2 * nt - (w.len - w.row0 - t * PK_ROWS <= PK_STEP);
    };
    auto next = [&](int k) {
        if (!wait(&B.work_full[k & 1], k >> 1)) return false;
        w = B.work[k & 1];
        if (w.len == 0) return false;
        n0 = w.row0 / PK_ROWS + 1;
        n1 = G::TILES > 1 && a.item_rows > PK_ROWS && w.len > w.row0 + PK_ROWS ? n0 + 1 : 0;
        n = G::STEPS == 2 ? max(n0, n1) : steps(0);
        return true;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PK_OTHER_REGS));
        if (warp == 10 && lane == 0) {
            // ---- loads: Q_0, K_0, Q_1, then V and K ----
            auto load = [&](uint8_t *dst, const CUtensorMap *map, int rows, int head, int row, uint64_t *bar) {
                mbar_arrive_expect_tx(bar, rows * HD * 2);
#pragma unroll
                for (int x = 0; x < HD; x += 64) pk_tma_load(dst + x / 64 * (rows * 128), map, x, head, row, bar);
            };
            int q[2] = {0, 0}, slot = 0, phase = 0, ahead = 0;   // Q tiles loaded, ring position, its tiles loaded in all
            for (int k = 0; next(k); ++k) {
                const int kvh = w.head / a.group;
                auto load_q = [&](int t) {
                    if (q[t] > 0 && !wait(&B.q_empty[t], q[t] + 1)) return;
                    load(sq + t * G::Q_TILE, &qmap, PK_ROWS, w.head, w.first + w.row0 + t * PK_ROWS, &B.q_full[t]);
                    ++q[t];
                };
                load_q(0);
                for (int i = 0; i < 2 * n && ok; ++i) {
                    if (!wait(&B.kv_empty[slot], phase + 1)) break;
                    int j;
                    const bool v = pk_is_value<G::STEPS>(i, n, j);
                    load(skv + slot * G::KV_TILE, v ? &vmap : &kmap, G::KEYS, kvh, w.first + j * G::KEYS, &B.kv_full[slot]);
                    ++ahead;
                    if (++slot == PK_STAGES) slot = 0, phase ^= 1;
                    if (i == 0 && n1) load_q(1);
                }
                mbar_arrive(&B.work_empty[k & 1]);
            }
            if (!ok) {   // the loads in flight land before the CTA leaves
                for (int k = max(0, ahead - PK_STAGES); k < ahead; ++k)
                    mbar_wait_bounded(&B.kv_full[k % PK_STAGES], k / PK_STAGES & 1, a.status, HOLO_E_TIMEOUT);
                for (int t = 0; t < 2; ++t)
                    if (q[t] > 0) mbar_wait_bounded(&B.q_full[t], (q[t] - 1) & 1, a.status, HOLO_E_TIMEOUT);
            }
        } else if (warp < 10) {
            // ---- MMAs of tile t ----
            // The whole warp walks the items together, so that the descriptors stay uniform (a thread of its own would
            // move each into uniform registers, at about the cost of the MMA); one lane issues.
            constexpr uint32_t id_s = tc_idesc_f16(PK_ROWS, PK_STEP) | PkType<T>::AB;
            constexpr uint32_t id_o = tc_idesc_f16(PK_ROWS, HD) | PkType<T>::AB | 1u << 16;   // B transposed
            constexpr uint32_t HALF = PK_STEP * 128 >> 4;   // 64 rows of a 128-byte-wide tile, in a descriptor
            const int t = warp - 8;
            const bool leader = pk_elect();
            const uint32_t sq_at = __shfl_sync(0xffffffffu, smem_addr(sq) >> 4, 0), skv_at = sq_at + (G::TILES * G::Q_TILE >> 4);
            int q = 0, it = 0;                     // Q tiles, steps so far
            int slot = 0, phase = 0;               // of the next ring tile
            auto wait_all = [&](uint64_t *bar, int parity) {
                wait(bar, parity);
                ok = __all_sync(0xffffffffu, ok);
                return ok;
            };
            auto commit = [&](uint64_t *bar) {
                if (leader) tc_commit(bar);
            };
            auto advance = [&]() {
                if (++slot == PK_STAGES) slot = 0, phase ^= 1;
            };
            // S of step x of all: Q_t and part h of the K tile in slot kv
            auto scores = [&](int x, int kv, int h) {
                tc_fence_after();
                const uint64_t qd = PK_DESC_K | (uint64_t)(sq_at + t * (G::Q_TILE >> 4));
                const uint64_t kd = PK_DESC_K | (uint64_t)(skv_at + kv * (G::KV_TILE >> 4) + h * HALF);
                if (leader) {
#pragma unroll
                    for (int s = 0; s < HD / 16; ++s) {
                        const uint64_t qo = (uint64_t)(((s >> 2) * (PK_ROWS * 128) + (s & 3) * 32) >> 4);
                        const uint64_t ko = (uint64_t)(((s >> 2) * (G::KEYS * 128) + (s & 3) * 32) >> 4);
                        tc_mma(t * 128 + (x & 1) * PK_STEP, qd + qo, kd + ko, id_s, s > 0);
                    }
                    tc_commit(&B.s_full[t][x & 1]);
                }
                __syncwarp();
            };
            for (int k = 0; ok; ++k) {
                const bool more = next(k);
                if (!__all_sync(0xffffffffu, more)) break;
                const int ns = __shfl_sync(0xffffffffu, steps(t), 0), tiles = __shfl_sync(0xffffffffu, n, 0);
                int k_slot = 0, v_slot = 0;
                // the ring's tiles in the order of their loads
                if (ns > 0) {
                    if (!wait_all(&B.q_full[t], q++) || !wait_all(&B.kv_full[slot], phase)) break;
                    k_slot = slot;
                    // the S that these write were read, as P, by the last steps of the item before
                    if (it > 1 && !wait_all(&B.o_done[t][it & 1], (it >> 1) + 1)) break;
                    scores(it, k_slot, 0);
                    if (ns > 1) {
                        if (G::STEPS == 1) {
                            commit(&B.kv_empty[k_slot]);
                            advance();
                            if (!wait_all(&B.kv_full[slot], phase)) break;
                            k_slot = slot;
                        }
                        if (it > 0 && !wait_all(&B.o_done[t][(it + 1) & 1], ((it + 1) >> 1) + 1)) break;
                        scores(it + 1, k_slot, G::STEPS - 1);
                    }
                    commit(&B.kv_empty[k_slot]);
                    if (ns <= 2) commit(&B.q_empty[t]);
                    advance();
                }
                for (int x = 0; x < ns && ok; ++x, ++it) {
                    const int h = x & (G::STEPS - 1);
                    const bool last = h == G::STEPS - 1;   // of its ring tile
                    if (h == 0) {
                        v_slot = slot;
                        if (!wait_all(&B.kv_full[v_slot], phase)) break;
                        if (w.careful && !wait_all(&B.kv_checked[v_slot], phase)) break;
                        advance();
                    }
                    if (!wait_all(&B.p_full[t][it & 1], it >> 1)) break;
                    tc_fence_after();
                    const uint64_t v = pk_desc_mn(G::KEYS) | (uint64_t)(skv_at + v_slot * (G::KV_TILE >> 4) + h * HALF);
                    if (leader) {
#pragma unroll
                        for (int s = 0; s < PK_STEP / 16; ++s)   // 16 keys: 8 columns of P, 16 rows of V
                            tc_mma_ts(256 + t * 128, t * 128 + (it & 1) * PK_STEP + 8 * s, v + (uint64_t)(s * 2048 >> 4), id_o,
                                      x > 0 || s > 0);
                        tc_commit(&B.o_done[t][it & 1]);
                        if (last || x + 1 == ns) tc_commit(&B.kv_empty[v_slot]);
                    }
                    __syncwarp();
                    if (x + 2 < ns) {
                        if (h == 0) {
                            k_slot = slot;
                            if (!wait_all(&B.kv_full[k_slot], phase)) break;
                            advance();
                        }
                        // P of this step and the next S but one share columns: P has been read first
                        if (!wait_all(&B.o_done[t][it & 1], it >> 1)) break;
                        scores(it, k_slot, h);
                        if (last || x + 3 == ns) commit(&B.kv_empty[k_slot]);
                        if (x + 3 == ns) commit(&B.q_empty[t]);
                    }
                }
                // tiles that only the other query tile reads
                for (int i = 2 * ((ns + G::STEPS - 1) / G::STEPS); i < 2 * tiles && ok; ++i) {
                    if (!wait_all(&B.kv_full[slot], phase)) break;
                    if (leader) mbar_arrive(&B.kv_empty[slot]);
                    advance();
                }
                if (lane == 0) mbar_arrive(&B.work_empty[k & 1]);
            }
            if (!ok) {   // the MMAs in flight end before the CTA leaves
                commit(&B.drain[t]);
                mbar_wait_bounded(&B.drain[t], 0, a.status, HOLO_E_TIMEOUT);
            }
        } else if (warp == 11) {
            // ---- items: every gridDim.x-th, the order turned round each time so that the sums are even ----
            int kept[PK_KEPT], first0 = 0;
            kept[0] = 0;
            if (lane < a.n_seqs) packed_seq(a, lane, first0, kept[0]);
#pragma unroll
            for (int i = 1; i < PK_KEPT; ++i) kept[i] = pk_len(a, 32 * i + lane);
            int published = 0, base = 0;           // items so far, and of them before this pass
            bool more = true;
            int careful = 0;
            auto publish = [&](PkWork &mine) {
                if (published >= 2) wait(&B.work_empty[published & 1], (published >> 1) + 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                mine.careful = careful;
                if (lane == 0) {
                    B.work[published & 1] = mine;
                    mbar_arrive(&B.work_full[published & 1]);
                }
                __syncwarp();
                ++published;
            };
            auto find = [&]() {
                if (!more) return;
                const int round = published - base;
                const long long r = (long long)round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                const int tile = (int)(r / a.n_heads);
                PkWork mine;
                mine.head = (int)(r - (long long)tile * a.n_heads);
                more = pk_find_work(a, kept, first0, tile, mine);   // past the end: none follows
                if (more) publish(mine);
            };
            find();
            find();
            int slot = 0, phase = 0;
            for (int k = 0; ok; ++k) {
                if (k == published) {
                    // The end of a pass.  Once the last item is through: is one with more care wanted?
                    if (k > 0 && careful < 2) {
                        wait(&B.work_empty[(k - 1) & 1], (k - 1) >> 1);
                        ok = __all_sync(0xffffffffu, ok);
                        const int again = *(volatile int *)&B.again;
                        if (ok && again > careful) {
                            careful = again;
                            more = true;
                            base = published;
                            find();
                            find();
                        }
                    }
                    if (k == published) {
                        PkWork none = {0, 0, 0, 0, 0};
                        publish(none);
                        break;
                    }
                }
                if (!next(k)) break;
                if (w.careful) {                // the rows of the item before have been written
                    wait(&B.work_empty[(k - 1) & 1], (k - 1) >> 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    for (int i = lane; i < PK_KINDS * HD; i += 32) (&seen[0][0])[i] = PK_NEVER;
                    __syncwarp();
                }
                for (int i = 0; i < 2 * n; ++i) {   // every tile of the ring, so that no phase is missed
                    wait(&B.kv_full[slot], phase);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    int j;
                    if (pk_is_value<G::STEPS>(i, n, j) && w.careful) {
                        uint8_t *tile = skv + slot * G::KV_TILE;
                        pk_clean_tile<T, HD, G::KEYS>(tile, j * G::KEYS - w.row0, w.len - w.row0, w.careful == 2, seen);
                        holo_mv::fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (lane == 0) {
                        mbar_arrive(&B.kv_checked[slot]);
                        mbar_arrive(&B.kv_empty[slot]);
                    }
                    if (++slot == PK_STAGES) slot = 0, phase ^= 1;
                }
                if (lane == 0) mbar_arrive(&B.bad_known[k & 1]);
                if (ok) find();
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PK_SOFTMAX_REGS));
        const int t = warp >> 2, r = threadIdx.x & 127;   // tile, row of the tile
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + t * 128 + lanes, to = tmem + 256 + t * 128 + lanes;
        const float c = a.scale * 1.4426950408889634f;
        int it = 0;                        // steps so far
        // a wait of the whole warp
        auto wait_warp = [&](uint64_t *bar, int parity) {
            wait(bar, parity);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            return ok;
        };
        for (int k = 0;; ++k) {
            const bool more = next(k);
            if (!__all_sync(0xffffffffu, more)) break;
            const int ns = steps(t);
            float m = -INFINITY;           // log2 of what P is scaled by
            float l = 0.0f;
            for (int x = 0; x < ns; ++x, ++it) {
                const uint32_t tb = ts + (it & 1) * PK_STEP;
                if (!wait_warp(&B.s_full[t][it & 1], it >> 1)) break;
                uint32_t s[PK_STEP];
                tc_ld64(tb, s);
                // the diagonal: row r sees keys 0 .. r of the tile
                const int seen = r - (x * PK_STEP - (t ? n1 - 1 : n0 - 1) * PK_ROWS);
                if (x / 2 == (t ? n1 : n0) - 1) {
#pragma unroll
                    for (int i = 0; i < PK_STEP; ++i)
                        if (i > seen) s[i] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < PK_STEP; i += 2)
                    top[i / 2 & 3] = pk_max3(top[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                const float mn = fmaxf(m, pk_max3(fmaxf(top[0], top[1]), top[2], top[3]) * c);
                const bool grow = mn > m + PK_GROWTH;
                if (x == 0) {
                    m = mn;
                } else if (__any_sync(0xffffffffu, grow)) {
                    const float fix = grow ? pk_ex2(m - mn) : 1.0f;
                    if (grow) m = mn;
                    l *= fix;
                    if (!wait_warp(&B.o_done[t][(it + 1) & 1], (it - 1) >> 1)) break;   // of the step before
#pragma unroll 1
                    for (int cb = 0; cb < HD; cb += 32) {
                        uint32_t o[32];
                        tc_ld32(to + cb, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                        tc_st32(to + cb, o);
                    }
                }
                const float sub = (m == -INFINITY ? 0.0f : m) - PkType<T>::LIFT;   // nothing but -inf so far: weights 0
                const uint64_t c2 = pk_pair(c, c), sub2 = pk_pair(-sub, -sub);
                uint64_t sum[2] = {0, 0};
                uint32_t p[PK_STEP / 2];
#pragma unroll
                for (int i = 0; i < PK_STEP / 2; ++i) {
                    const uint64_t z = pk_fma2(pk_pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, sub2);
                    float y0, y1;
                    pk_split(z, y0, y1);
                    y0 = pk_ex2(y0);
                    y1 = pk_ex2(y1);
                    sum[i & 1] = pk_add2(sum[i & 1], pk_pair(y0, y1));
                    p[i] = PkType<T>::pack(y0, y1);
                }
                tc_st32(tb, p);
                tc_fence_before();
                mbar_arrive(&B.p_full[t][it & 1]);
                float y0, y1;
                pk_split(pk_add2(sum[0], sum[1]), y0, y1);
                l += y0 + y1;
            }
            if (!ok) break;
            // ---- O_t / l to the rows ----
            if (ns > 0) {
                if (w.careful) wait(&B.bad_known[k & 1], k >> 1);
                if (!wait_warp(&B.o_done[t][(it + 1) & 1], (it - 1) >> 1)) break;
                const int i = w.row0 + t * PK_ROWS + r;   // of the sequence
                const float inv = w.careful == 2 ? 1.0f / PK_DOWN / l : 1.0f / l;
                bool finite = true;            // all of the sums
                // 32 values a lane at a time; four lanes turn their 16-byte pieces round, so that they store 64 bytes of a row
                const int part = lane & 3, i4 = i - part, n4 = w.len - i4;   // the first row of the four, rows from it on
                T *o = (T *)a.out + (size_t)(w.first + min(i4, w.len - 1)) * a.out_row + (size_t)w.head * a.out_head + 8 * part;
#pragma unroll (HD == 256 ? 2 : HD / 32)
                for (int cb = 0; cb < HD; cb += 32) {
                    uint32_t v[32];
                    tc_ld32(to + cb, v);
                    uint32_t u[4][4];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float x = __uint_as_float(v[2 * e]) * inv, y = __uint_as_float(v[2 * e + 1]) * inv;
                        finite = finite && isfinite(x) && isfinite(y);
                        u[e >> 2][e & 3] = PkType<T>::pack(x, y);
                    }
#pragma unroll
                    for (int bit = 1; bit < 4; bit <<= 1)
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            if (!(p & bit)) {
                                const bool up = (lane & bit) != 0;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? u[p][e] : u[p | bit][e], bit);
                                    if (up) u[p][e] = got;
                                    else u[p | bit][e] = got;
                                }
                            }
#pragma unroll
                    for (int p = 0; p < 4; ++p)
                        if (p < n4) *reinterpret_cast<uint4 *>(o + p * a.out_row + cb) = make_uint4(u[p][0], u[p][1], u[p][2], u[p][3]);
                }
                __syncwarp();              // a row is written by four lanes
                if (i < w.len) {
                    if (!w.careful) {
                        if (!finite) atomicMax(&B.again, 1);
                    } else if (l > 0.0f && l < INFINITY) {   // else its scores have made the row NaN
                        // finite weights and values whose sums are not have overflowed (fp16's cannot)
                        if (std::is_same<T, __nv_bfloat16>::value && !finite) atomicMax(&B.again, 2);
                        pk_mark_row<T, HD>((T *)a.out + (size_t)(w.first + i) * a.out_row + (size_t)w.head * a.out_head,
                                           t * PK_ROWS + r, seen);
                    }
                    if (a.lse) a.lse[(size_t)w.head * a.total + w.first + i] = (m - PkType<T>::LIFT + log2f(l)) * 0.6931471805599453f;
                }
                __syncwarp();
            }
            tc_fence_before();             // O_t has been read before the next item's P_t is announced
            if (lane == 0) mbar_arrive(&B.work_empty[k & 1]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tc_dealloc(tmem, PK_TMEM_COLS);
    }
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
EncodeTiled encode_tiled() {
    static std::once_flag once;
    static EncodeTiled fn = nullptr;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = (EncodeTiled)p;
        cudaGetLastError();
    });
    return fn;
}

// [rows][heads][hd] as boxes of `tall` rows of one head, 64 values wide; rows past
// the end read as zeros.  A stride that one row or head leaves open is any valid one.
bool make_map(CUtensorMap *map, int type, const void *p, int hd, int heads, int rows, long long row, long long head,
              int tall) {
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)row * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)tall}, one[3] = {1, 1, 1};
    const CUtensorMapDataType dt = type == HOLO_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode_tiled()(map, dt, 3, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
bool launch_tc(const PackedArgs &a, int type, cudaStream_t st) {
    CUtensorMap qm, km, vm;
    const int kv = a.n_heads / a.group;
    if (!make_map(&qm, type, a.q, HD, a.n_heads, a.total, a.q_row, a.q_head, PK_ROWS) ||
        !make_map(&km, type, a.k, HD, kv, a.total, a.k_row, a.k_head, PkGeom<HD>::KEYS) ||
        !make_map(&vm, type, a.v, HD, kv, a.total, a.v_row, a.v_head, PkGeom<HD>::KEYS))
        return false;
    static bool configured[16] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 16 || !configured[dev]) {
        if (cudaFuncSetAttribute(packed_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)PkGeom<HD>::SMEM) != cudaSuccess)
            return false;
        if (dev < 16) configured[dev] = true;
    }
    // at most this many items; where pairs of tiles would leave SMs without one, single tiles
    PackedArgs w = a;
    const int sms = holo_dev()->sms;
    auto items = [&](int rows) { return ((long long)a.total + (long long)(rows - 1) * a.n_seqs) / rows * a.n_heads; };
    w.item_rows = PkGeom<HD>::TILES == 2 && items(2 * PK_ROWS) >= sms ? 2 * PK_ROWS : PK_ROWS;
    const unsigned grid = (unsigned)min((long long)sms, items(w.item_rows));
    return holo_launch_early(packed_tc_kernel<T, HD>, grid, PK_THREADS, PkGeom<HD>::SMEM, st, w, qm, km, vm) == cudaSuccess;
}

template <typename T>
bool launch_tc(const PackedArgs &a, int hd, int type, cudaStream_t st) {
    return hd == 64 ? launch_tc<T, 64>(a, type, st) : hd == 128 ? launch_tc<T, 128>(a, type, st) : launch_tc<T, 256>(a, type, st);
}

// whether TMA can address rows of this base and these strides (elements)
bool tma_rows(const void *p, long long row, long long head) {
    return (uintptr_t)p % 16 == 0 && row % 8 == 0 && head % 8 == 0 && row < (1LL << 38) && head < (1LL << 38);
}

}  // namespace

extern "C" int cuda_attention_packed(const holo_packed_desc *d, void *out, const void *q, const void *k, const void *v,
                                     const int *cu_seqlens, float *lse) {
    const char *what = "cuda_attention_packed";
    HoloDevice *D = holo_dev();
    if (!D) return cuda_last_status();
    auto refuse = [&](int code) {
        holo_set_status(code, what);
        return code;
    };
    if (!d || d->n_heads <= 0 || d->n_kv_heads <= 0 || d->n_heads % d->n_kv_heads || d->n_seqs < 0 || d->total < 0 ||
        !(d->scale >= 0.0f))
        return refuse(HOLO_E_ARG);
    if ((d->type != HOLO_DT_F16 && d->type != HOLO_DT_BF16) || (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) ||
        d->n_heads > 65535)
        return refuse(HOLO_E_UNSUPPORTED);
    if (d->total == 0) return HOLO_OK;
    if (!out || !q || !k || !v || !cu_seqlens || d->n_seqs == 0 ||
        ((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 2)
        return refuse(HOLO_E_ARG);
    const long long hd = d->head_dim;
    PackedArgs a;
    a.out = out, a.q = q, a.k = k, a.v = v, a.cu = cu_seqlens, a.lse = lse;
    a.n_seqs = d->n_seqs, a.total = d->total, a.n_heads = d->n_heads, a.group = d->n_heads / d->n_kv_heads;
    a.scale = d->scale == 0.0f ? 1.0f / sqrtf((float)hd) : d->scale;
    a.q_row = d->q_row ? d->q_row : d->n_heads * hd, a.q_head = d->q_head ? d->q_head : hd;
    a.k_row = d->k_row ? d->k_row : d->n_kv_heads * hd, a.k_head = d->k_head ? d->k_head : hd;
    a.v_row = d->v_row ? d->v_row : d->n_kv_heads * hd, a.v_head = d->v_head ? d->v_head : hd;
    a.out_row = d->out_row ? d->out_row : d->n_heads * hd, a.out_head = d->out_head ? d->out_head : hd;
    a.status = D->status;
    if (a.q_row < hd || a.k_row < hd || a.v_row < hd || a.out_row < hd || a.q_head < hd || a.k_head < hd || a.v_head < hd ||
        a.out_head < hd)
        return refuse(HOLO_E_ARG);
    cudaStream_t st = d->stream ? (cudaStream_t)d->stream : holo_stream();
    bool done = false;
    if (tma_rows(q, a.q_row, a.q_head) && tma_rows(k, a.k_row, a.k_head) && tma_rows(v, a.v_row, a.v_head) &&
        tma_rows(out, a.out_row, a.out_head) && encode_tiled())
        done = d->type == HOLO_DT_F16 ? launch_tc<__half>(a, d->head_dim, d->type, st)
                                      : launch_tc<__nv_bfloat16>(a, d->head_dim, d->type, st);
    if (!done) {
        if (d->type == HOLO_DT_F16) launch_simple<__half>(a, d->head_dim, st);
        else launch_simple<__nv_bfloat16>(a, d->head_dim, st);
    }
    return holo_check_launch(what) ? HOLO_OK : cuda_last_status();
}
