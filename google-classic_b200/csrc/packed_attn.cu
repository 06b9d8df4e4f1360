// packed_attn.cu -- causal attention of whole prompts of different lengths
// that lie one after another in the rows (holo_b200.h, cuda_attention_packed).
#include "holo_common.cuh"

#include <cuda_bf16.h>
#include <cfloat>

namespace {

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
};

// the sequence of a row: the last s with cu[s] <= row
__device__ __forceinline__ int packed_seq(const int *__restrict__ cu, int n, int row) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One warp a row and head, lane l holding dims l, l + 32, ...: online softmax
// over the row's own keys.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
packed_simple_kernel(const __grid_constant__ PackedArgs a) {
    constexpr int NB = HD / 32;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y, lane = threadIdx.x & 31;
    if (row >= a.total) return;
    const int s = packed_seq(a.cu, a.n_seqs, row);
    const int first = max(0, a.cu[s]);
    const T *q = (const T *)a.q + row * a.q_row + h * a.q_head;
    float qv[NB], acc[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        qv[b] = to_float(q[32 * b + lane]) * a.scale;
        acc[b] = 0.0f;
    }
    for (int j = first; j <= row; ++j) {
        const T *k = (const T *)a.k + j * a.k_row + h / a.group * a.k_head, *v = (const T *)a.v + j * a.v_row + h / a.group * a.v_head;
        float dot = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) dot = fmaf(qv[b], to_float(k[32 * b + lane]), dot);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float mn = fmaxf(m, dot), fix = expf(m - mn), e = expf(dot - mn);
        l = l * fix + e;
        m = mn;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = fmaf(e, to_float(v[32 * b + lane]), acc[b] * fix);
    }
    T *o = (T *)a.out + row * a.out_row + h * a.out_head;
#pragma unroll
    for (int b = 0; b < NB; ++b) from_float(acc[b] / l, o[32 * b + lane]);
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

}  // namespace

extern "C" int cuda_attention_packed(const holo_packed_desc *d, void *out, const void *q, const void *k, const void *v,
                                     const int *cu_seqlens, float *lse) {
    const char *what = "cuda_attention_packed";
    if (!holo_dev()) return cuda_last_status();
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
    if (a.q_row < hd || a.k_row < hd || a.v_row < hd || a.out_row < hd || a.q_head < hd || a.k_head < hd || a.v_head < hd ||
        a.out_head < hd)
        return refuse(HOLO_E_ARG);
    cudaStream_t st = d->stream ? (cudaStream_t)d->stream : holo_stream();
    if (d->type == HOLO_DT_F16) launch_simple<__half>(a, d->head_dim, st);
    else launch_simple<__nv_bfloat16>(a, d->head_dim, st);
    return holo_check_launch(what) ? HOLO_OK : cuda_last_status();
}
