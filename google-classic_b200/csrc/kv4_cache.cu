// kv4_cache.cu -- the paged 4-bit KV cache: sizes and argument checks, rows of
// keys and values quantised into their pages, and read back.
//
// Four lanes hold a group of 32 values (eight each) of one row, head and side:
// the group's value of largest magnitude is found over them with shuffles, and
// a lane writes the word of its eight key codes, or two halfwords of value codes.
// A CTA takes up to 16 rows, whose places (sequence, page, block) are looked up
// once; rows that share a block meet in one CTA, so its partly written sectors are
// completed in L2.  Both kernels move each byte once.  Few rows are bound by
// latency (of the look-ups, the loads and the call); many, 36,829 of 8 heads of 128
// in fp16, take 64 us to write (3.0 TB/s), bound by the quantiser's instructions, and
// 40 us to read (4.8 TB/s), by the look-ups at a CTA's start and the stores.  More rows a CTA
// (32, 64) or more rows' loads together in the read (2, 4) gained nothing.
#include "kv4.cuh"

#include <mutex>
#include <type_traits>

namespace {

constexpr int ROW_THREADS = 256;

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t counter_bytes(const holo_kv4 *c) {
    return round256(sizeof(int) * (size_t)c->max_seqs * c->n_kv_heads * (KV4_MAX_GROUP / KV4_HEADS));
}
size_t plan_bytes(const holo_kv4 *c) { return round256(sizeof(int) * (16 + 3 * (size_t)c->n_pages + 2 * (size_t)c->max_seqs)); }
size_t partial_bytes(const holo_kv4 *c) {
    return sizeof(float) * (size_t)KV4_MAX_CTAS * 2 * KV4_HEADS * (c->head_dim + 2);
}

std::mutex g_work_mu;

// Device memory, zero, without touching a stream of anyone's: also while one is being captured.
void *zero_memory(size_t size) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // of this thread, until it is put back
    cudaThreadExchangeStreamCaptureMode(&mode);
    void *p = nullptr;
    cudaStream_t st = nullptr;
    const bool done = cudaMalloc(&p, size) == cudaSuccess && cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) == cudaSuccess &&
                      cudaMemsetAsync(p, 0, size, st) == cudaSuccess && cudaStreamSynchronize(st) == cudaSuccess;
    if (st) cudaStreamDestroy(st);
    if (!done) {
        cudaGetLastError();
        cudaFree(p);
        p = nullptr;
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    return p;
}

// A buffer of the library's own on the current device, zero when it is made.  One
// that is too small is kept, since calls under way and captured graphs may hold it; sizes
// are powers of two, so that all that were outgrown are no larger than the last.
bool own_buffer(HoloDevice *D, void *&buf, size_t &have, size_t bytes) {
    if (have >= bytes) return true;
    size_t size = 1 << 16;
    while (size < bytes) size *= 2;
    void *p = zero_memory(size);
    if (!p) {
        holo_set_status(HOLO_E_NOMEM, "kv4 workspace");
        return false;
    }
    if (buf) D->kv4_outgrown.push_back(buf);
    buf = p;
    have = size;
    return true;
}

// The library's own workspace.  Caches of all shapes use it in turn, so the counters, which have to be zero before a
// call, have a buffer that nothing else is written to; no call reads what another left in the other sections.
bool own_work(HoloDevice *D, const holo_kv4 *c, Kv4Work *work) {
    std::lock_guard<std::mutex> lk(g_work_mu);
    if (!own_buffer(D, D->kv4_counters, D->kv4_counter_bytes, counter_bytes(c)) ||
        !own_buffer(D, D->kv4_work, D->kv4_work_bytes, plan_bytes(c) + partial_bytes(c)))
        return false;
    work->counters = (int *)D->kv4_counters;
    work->plan = (int *)D->kv4_work;
    work->partial = (float *)((uint8_t *)D->kv4_work + plan_bytes(c));
    return true;
}

// the sequence i with cu[i] <= row < cu[i + 1]: the last i with cu[i] <= row
__device__ __forceinline__ int seq_of_row(const int *cu, int n, int row) {
    int lo = 0, hi = n;   // cu[lo] <= row < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(cu + mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

constexpr int ROW_MAX = 16;            // rows a CTA

// where a row lies: byte offset of its block of KV head 0 in the layer (-1:
// nowhere), place in the block
struct Place {
    long long at;
    int slot;
};

__device__ __forceinline__ Place row_place(const Kv4View &c, int hd, const int *cu, const int *start, const int *seqs,
                                           int n, int row) {
    const int i = seq_of_row(cu, n, row);
    const int first = __ldcg(cu + i), end = __ldcg(cu + i + 1), at0 = __ldcg(start + i), s = seqs ? __ldcg(seqs + i) : i;
    Place p = {-1, 0};
    if (row < first || row >= end || at0 < 0) return p;
    const long long pos = (long long)at0 + (row - first);
    if (s < 0 || s >= c.max_seqs || pos >= (long long)c.max_pages * c.page_tokens) {
        kv4_report(c.status, HOLO_E_ARG);
        return p;
    }
    const int col = (int)pos / c.page_tokens, in_page = (int)pos - col * c.page_tokens;
    const int page = __ldcg(c.tables + (size_t)s * c.max_pages + col);
    if (page < 0 || page >= c.n_pages) {
        kv4_report(c.status, HOLO_E_ARG);
        return p;
    }
    p.at = ((long long)page * c.n_kv * c.page_blocks + in_page / KV4_BLOCK) * kv4_block_bytes(hd);
    p.slot = in_page % KV4_BLOCK;
    return p;
}

// eight values of a row; wide: 16-byte aligned
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool wide, float (&x)[8]) {
    if (wide) {
        uint4 w[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldcg(reinterpret_cast<const uint4 *>(p) + i);
        const T *h = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kv4_to_float<T>(h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kv4_to_float<T>(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, bool wide, const T (&x)[8]) {
    if (wide) {
        uint4 w[sizeof(T) / 2];
        T *h = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = x[i];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
}

// Eight codes of a lane and the scale of its group, over the four lanes that
// hold it: d = fp16(m / -8), code = rint(x / d) + 8 in 0..15 (fp32 arithmetic,
// each operation rounded once), NaN as the scale where a value is not finite or
// the scale would be infinite (its product with a zero that a sum leaves is not always NaN).
// Bound by instructions (an append of many rows: 0.79 of the issue slots), so the work is put on the FMA pipe, which takes one a cycle:
//   m         from the group's largest and smallest value; where they are equal
//             in size, or zero, from a second look for the first of them
//   x / d     the rounded quotient without a division: from the rounded
//             reciprocal r, t = x r and t + (x - t d) r, fused operations, which
//             rounds x / d correctly (Markstein, IBM J. Res. Dev. 34, 1990); where
//             the remainder could underflow the quotient is far below 1/2
//   codes     rounded to whole numbers by adding and taking away 1.5 * 2^23, and
//             put together four at a time as the digits, base 16, of an exact float
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], __half &d) {
    float high = x[0], low = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(high) : "f"(x[i]));
        low = fminf(low, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float h = __shfl_xor_sync(0xffffffffu, high, o), l = __shfl_xor_sync(0xffffffffu, low, o);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(high) : "f"(h));
        low = fminf(low, l);
    }
    float m = high > -low ? high : low;
    const bool tie = high == -low;
    if (__any_sync(0xffffffffu, tie)) {
        // the first value of that size: its place in the group, and the value
        int place = 32;
        float v = m;
#pragma unroll
        for (int i = 7; i >= 0; --i)
            if (fabsf(x[i]) == high) place = (threadIdx.x & 3) * 8 + i, v = x[i];
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const int p = __shfl_xor_sync(0xffffffffu, place, o);
            const float u = __shfl_xor_sync(0xffffffffu, v, o);
            if (p < place) place = p, v = u;
        }
        if (tie) m = v;
    }
    const bool finite = high < INFINITY && low > -INFINITY;   // high is NaN where a value is
    d = finite ? __float2half_rn(m * -0.125f) : __ushort_as_half(0x7e00);
    const float w = __half2float(d);
    const bool usable = w != 0.0f && fabsf(w) <= 65504.0f;   // a scale to divide by: else code 8
    if (!(fabsf(w) <= 65504.0f)) d = __ushort_as_half(0x7e00);
    const float r = usable ? __frcp_rn(w) : 0.0f;
    const float magic = 12582912.0f;
    uint32_t codes[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float digits = 0.0f;
#pragma unroll
        for (int i = 4 * half + 3; i >= 4 * half; --i) {
            const float t = __fmul_rn(x[i], r);
            const float q = fminf(fmaxf(fmaf(fmaf(-t, w, x[i]), r, t), -8.0f), 7.0f);
            digits = fmaf(digits, 16.0f, __fadd_rn(__fadd_rn(q, magic), 8.0f - magic));
        }
        codes[half] = __float_as_uint(__fadd_rn(digits, 8388608.0f));   // 2^23: the digits are the low bits
    }
    return usable ? __byte_perm(codes[0], codes[1], 0x5410) : 0x88888888u;
}

// pair p (0..3) of eight codes, p and p + 4, as fp16 code - 8: 1024 + code, less 1032
__device__ __forceinline__ __half2 code_pair(uint32_t codes, int p) {
    const uint32_t w = (codes >> (4 * p) & 0x000f000fu) | 0x64006400u;
    return __hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6408)));
}

// the values of eight codes, rounded once to the rows' type
template <typename T>
__device__ __forceinline__ void dequantise8(uint32_t codes, __half d, T (&x)[8]) {
    const float w = __half2float(d);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const __half2 c = code_pair(codes, p);
        if constexpr (std::is_same<T, __half>::value) {   // the product has 15 bits: one rounding here too
            const __half2 v = __hmul2(c, __half2half2(d));
            x[p] = __low2half(v), x[p + 4] = __high2half(v);
        } else {
            const float2 v = __half22float2(c);
            x[p] = kv4_from_float<T>(v.x * w), x[p + 4] = kv4_from_float<T>(v.y * w);
        }
    }
}

// Thread = (row, head, group b, eight values t), of the CTA's rows.  A row is
// `lanes` = n_kv * HD / 8 threads; 1 << shift of them, the largest power of two in
// it, stand side by side, so that a thread keeps its place in the row from row to row.
template <bool APPEND, typename T, int HD>
__global__ void __launch_bounds__(ROW_THREADS)
rows_kernel(const __grid_constant__ Kv4View c, T *k, T *v, long long k_row, long long v_row, int rows, const int *cu,
            const int *start, const int *seqs, int n, bool wide, int rows_cta, int lanes, int shift) {
    constexpr int NB = HD / KV4_GROUP, EIGHTS = HD / 8;
    __shared__ Place places[ROW_MAX];
    early_wait();
    early_next();
    const int row0 = blockIdx.x * rows_cta, mine = min(rows_cta, rows - row0);
    if ((int)threadIdx.x < mine) places[threadIdx.x] = row_place(c, HD, cu, start, seqs, n, row0 + threadIdx.x);
    __syncthreads();
    const int across = 1 << shift, down = ROW_THREADS >> shift, r0 = threadIdx.x >> shift;
    for (int col0 = blockIdx.y << shift; col0 < lanes; col0 += gridDim.y << shift) {
        const int col = col0 + (threadIdx.x & (across - 1));
        const int kvh = col / EIGHTS, eight = col % EIGHTS, b = eight >> 2, t = eight & 3;
        const long long off = (long long)kvh * c.page_blocks * kv4_block_bytes(HD);
        T *kp = k + (size_t)(row0 + r0) * k_row + 8 * col, *vp = v + (size_t)(row0 + r0) * v_row + 8 * col;
        // (all threads of the CTA go round alike: the shuffles)
        for (int i = 0; i < mine; i += down, kp += down * k_row, vp += down * v_row) {
            const bool in = i + r0 < mine;
            const Place p = places[in ? i + r0 : 0];
            const bool ok = in && p.at >= 0;
            uint8_t *blk = c.pool + (p.at + off);
            const int pair = p.slot >> 1, odd = p.slot & 1;
            uint32_t *word = reinterpret_cast<uint32_t *>(blk + kv4_k_half(HD, 0, 2 * t, b) + p.slot * (HD / 2));
            uint8_t *value = blk + kv4_off_v(HD) + kv4_v_half(HD, 0, 2 * t, b) + pair * (8 * NB) + odd * (2 * NB);
            uint16_t *half0 = reinterpret_cast<uint16_t *>(value), *half1 = reinterpret_cast<uint16_t *>(value + 4 * NB);
            __half *scale_k = reinterpret_cast<__half *>(blk + kv4_off_dk(HD) + 2 * b + p.slot * (2 * NB));
            __half *scale_v = scale_k + HD / 2;
            if (APPEND) {
                float xk[8] = {}, xv[8] = {};
                if (ok) {
                    load8(kp, wide, xk);
                    load8(vp, wide, xv);
                }
                __half dk, dv;
                const uint32_t ck = quantise8(xk, dk), cv = quantise8(xv, dv);
                if (ok) {
                    *word = ck;
                    *half0 = (uint16_t)cv;
                    *half1 = (uint16_t)(cv >> 16);
                    if (t == 0) *scale_k = dk, *scale_v = dv;
                }
            } else if (in) {
                // (a row without a place: code 8 throughout, zeros)
                const uint32_t ck = ok ? *word : 0x88888888u, cv = ok ? *half0 | (uint32_t)*half1 << 16 : 0x88888888u;
                const __half dk = ok ? *scale_k : __ushort_as_half(0), dv = ok ? *scale_v : __ushort_as_half(0);
                T xk[8], xv[8];
                dequantise8(ck, dk, xk);
                dequantise8(cv, dv, xv);
                store8(kp, wide, xk);
                store8(vp, wide, xv);
            }
        }
    }
}
static_assert(kv4_v_half(128, 0, 1, 0) == 4 * 4 && kv4_v_half(64, 3, 0, 0) == 8 * 2 + 2 * 2, "a value's place in its block");

int type_bytes(int type) { return type == HOLO_DT_F32 ? 4 : 2; }

struct Rows {
    const holo_kv4 *c;
    void *k, *v;
    long long k_row, v_row;
    int rows;
    const int *cu, *start, *seqs;
    int n;
};

template <bool APPEND, typename T, int HD>
void launch_rows(const Rows &r, const Kv4View &view, bool wide, int sms, cudaStream_t st) {
    // 16 rows a CTA where that still makes four CTAs an SM, else fewer, and the columns of
    // a row over several CTAs where one row is all there is for each SM
    const int lanes = view.n_kv * (HD / 8);
    const int rows_cta = max(1, min(ROW_MAX, r.rows / (4 * sms)));
    int shift = 3;                            // lanes is a multiple of eight
    while (shift < 8 && lanes % (2 << shift) == 0) ++shift;
    const unsigned x = (unsigned)((r.rows + rows_cta - 1) / rows_cta);
    const unsigned y = (unsigned)max(1, min(lanes >> shift, (int)(4 * sms / x)));
    holo_launch_early(rows_kernel<APPEND, T, HD>, dim3(x, y), ROW_THREADS, 0, st, view, (T *)r.k, (T *)r.v, r.k_row, r.v_row,
                      r.rows, r.cu, r.start, r.seqs, r.n, wide, rows_cta, lanes, shift);
}

template <bool APPEND, typename T>
void launch_rows_hd(const Rows &r, const Kv4View &view, bool wide, int sms, cudaStream_t st) {
    switch (r.c->head_dim) {
    case 64: launch_rows<APPEND, T, 64>(r, view, wide, sms, st); break;
    case 128: launch_rows<APPEND, T, 128>(r, view, wide, sms, st); break;
    default: launch_rows<APPEND, T, 256>(r, view, wide, sms, st); break;
    }
}

template <bool APPEND>
int run_rows(Rows r, int layer, int type, const char *what) {
    Kv4View view;
    cudaStream_t st;
    if (!kv4_begin(r.c, layer, what, view, st, nullptr)) return cuda_last_status();
    if (type != HOLO_DT_F32 && type != HOLO_DT_F16 && type != HOLO_DT_BF16) {
        holo_set_status(HOLO_E_UNSUPPORTED, what);
        return HOLO_E_UNSUPPORTED;
    }
    const long long dense = (long long)r.c->n_kv_heads * r.c->head_dim;
    if (r.k_row == 0) r.k_row = dense;
    if (r.v_row == 0) r.v_row = dense;
    if (r.rows < 0 || r.n < 0 || r.n > r.c->max_seqs || r.k_row < dense || r.v_row < dense ||
        (r.rows > 0 && r.n > 0 && (!r.k || !r.v || !r.cu || !r.start))) {
        holo_set_status(HOLO_E_ARG, what);
        return HOLO_E_ARG;
    }
    if (r.rows == 0 || r.n == 0) return HOLO_OK;
    const int size = type_bytes(type);
    if (((uintptr_t)r.k | (uintptr_t)r.v) % size) {
        holo_set_status(HOLO_E_ARG, what);
        return HOLO_E_ARG;
    }
    // 16-byte accesses where every eight values of a row are aligned, else one by one
    const bool wide = ((uintptr_t)r.k | (uintptr_t)r.v) % 16 == 0 && (r.k_row * size | r.v_row * size) % 16 == 0;
    const int sms = holo_dev()->sms;
    switch (type) {
    case HOLO_DT_F32: launch_rows_hd<APPEND, float>(r, view, wide, sms, st); break;
    case HOLO_DT_F16: launch_rows_hd<APPEND, __half>(r, view, wide, sms, st); break;
    default: launch_rows_hd<APPEND, __nv_bfloat16>(r, view, wide, sms, st); break;
    }
    return kv4_end(what);
}

}  // namespace

bool kv4_shape_ok(const holo_kv4 *c) {
    return c && c->n_layers > 0 && c->n_kv_heads > 0 && (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) &&
           c->page_tokens > 0 && c->page_tokens <= 256 && c->page_tokens % KV4_BLOCK == 0 && c->n_pages > 0 &&
           c->max_seqs > 0 && c->max_pages > 0 && c->n_kv_heads <= 1024 && c->max_seqs <= (1 << 16) &&
           c->n_pages <= (1 << 20) && (long long)c->max_pages * c->page_tokens <= 0x7fffffffLL;
}

bool kv4_begin(const holo_kv4 *c, int layer, const char *what, Kv4View &view, cudaStream_t &st, Kv4Work *work) {
    HoloDevice *D = holo_dev();
    if (!D) return false;
    if (!kv4_shape_ok(c) || layer < 0 || layer >= c->n_layers || !c->pool || (uintptr_t)c->pool % 16 || !c->tables ||
        !c->lens) {
        holo_set_status(HOLO_E_ARG, what);
        return false;
    }
    st = c->stream ? (cudaStream_t)c->stream : holo_stream();
    view.page_blocks = c->page_tokens / KV4_BLOCK;
    const size_t page = (size_t)c->n_kv_heads * view.page_blocks * kv4_block_bytes(c->head_dim);
    view.pool = (uint8_t *)c->pool + (size_t)layer * c->n_pages * page;
    view.tables = c->tables;
    view.lens = c->lens;
    view.refs = c->refs;
    view.n_kv = c->n_kv_heads;
    view.page_tokens = c->page_tokens;
    view.n_pages = c->n_pages;
    view.max_seqs = c->max_seqs;
    view.max_pages = c->max_pages;
    view.status = D->status;
    if (work && !c->work) return own_work(D, c, work);
    if (work) {
        uint8_t *w = (uint8_t *)c->work;
        if ((uintptr_t)w % 16) {
            holo_set_status(HOLO_E_ARG, what);
            return false;
        }
        work->counters = (int *)w;
        work->plan = (int *)(w + counter_bytes(c));
        work->partial = (float *)(w + counter_bytes(c) + plan_bytes(c));
    }
    return true;
}

int kv4_end(const char *what) { return holo_check_launch(what) ? HOLO_OK : cuda_last_status(); }

extern "C" {

size_t cuda_kv4_pool_bytes(const holo_kv4 *c) {
    if (!kv4_shape_ok(c)) return 0;
    return (size_t)c->n_layers * c->n_pages * c->n_kv_heads * (c->page_tokens / KV4_BLOCK) * kv4_block_bytes(c->head_dim);
}

size_t cuda_kv4_work_bytes(const holo_kv4 *c) {
    if (!kv4_shape_ok(c)) return 0;
    return counter_bytes(c) + plan_bytes(c) + partial_bytes(c);
}

int cuda_kv4_append(const holo_kv4 *c, int layer, const void *k, const void *v, int type, long long k_row,
                    long long v_row, int rows, const int *cu_rows, const int *start, const int *seqs, int n) {
    return run_rows<true>({c, (void *)k, (void *)v, k_row, v_row, rows, cu_rows, start, seqs, n}, layer, type,
                          "cuda_kv4_append");
}

int cuda_kv4_read(const holo_kv4 *c, int layer, void *k, void *v, int type, long long k_row, long long v_row, int rows,
                  const int *cu_rows, const int *start, const int *seqs, int n) {
    return run_rows<false>({c, k, v, k_row, v_row, rows, cu_rows, start, seqs, n}, layer, type, "cuda_kv4_read");
}

}  // extern "C"
