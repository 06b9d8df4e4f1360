// kv4_attn.cu -- attention of one query a sequence over the paged 4-bit cache.
#include "kv4.cuh"

#include <cfloat>

namespace {

constexpr int AT_WARPS = 8;

// CTA = one query head of one sequence: warps take every eighth position and
// keep their own running maximum, sum and weighted sum of values.
template <typename T, int HD>
__global__ void __launch_bounds__(AT_WARPS * 32)
kv4_attn_simple_kernel(const __grid_constant__ Kv4View c, T *__restrict__ out, const T *__restrict__ q, long long q_row,
                       long long out_row, int group, float scale, const int *__restrict__ seqs, int n) {
    constexpr int NB = HD / 32;   // lane l holds value l of every group
    const int h = blockIdx.x, i = blockIdx.y, kvh = h / group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int s = seqs ? seqs[i] : i;
    if (s < 0 || s >= c.max_seqs) {
        if (threadIdx.x == 0) kv4_report(c.status, HOLO_E_ARG);
        return;
    }
    const int len = c.lens[s];
    const int *table = c.tables + (size_t)s * c.max_pages;
    float qv[NB], acc[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        qv[b] = kv4_to_float<T>(q[i * q_row + h * HD + 32 * b + lane]) * scale;
        acc[b] = 0.0f;
    }
    for (int p = warp; p < len; p += AT_WARPS) {
        const int page = table[p / c.page_tokens];
        if (page < 0 || page >= c.n_pages) {
            if (lane == 0) kv4_report(c.status, HOLO_E_ARG);
            continue;
        }
        const int slot = p % KV4_BLOCK;
        const uint8_t *blk = kv4_block(c, HD, page, kvh, p % c.page_tokens / KV4_BLOCK);
        float dot = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int code = *reinterpret_cast<const uint16_t *>(blk + kv4_k_half(HD, slot, lane >> 2, b)) >> (4 * (lane & 3)) & 15;
            const float d = __half2float(*reinterpret_cast<const __half *>(blk + kv4_off_dk(HD) + 2 * (slot * NB + b)));
            dot = fmaf(qv[b], d * (float)(code - 8), dot);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float mn = fmaxf(m, dot), fix = expf(m - mn), e = expf(dot - mn);
        l = l * fix + e;
        m = mn;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int code = *reinterpret_cast<const uint16_t *>(blk + kv4_off_v(HD) + kv4_v_half(HD, slot, lane >> 2, b)) >>
                             (4 * (lane & 3)) & 15;
            const float d = __half2float(*reinterpret_cast<const __half *>(blk + kv4_off_dv(HD) + 2 * (slot * NB + b)));
            acc[b] = acc[b] * fix + e * (d * (float)(code - 8));
        }
    }
    __shared__ float sm[AT_WARPS], sl[AT_WARPS], sa[AT_WARPS][HD];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int b = 0; b < NB; ++b) sa[warp][32 * b + lane] = acc[b];
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < AT_WARPS; ++w) top = fmaxf(top, sl[w] == 0.0f ? -INFINITY : sm[w]);
    for (int d = threadIdx.x; d < HD; d += AT_WARPS * 32) {
        float sum = 0.0f, all = 0.0f;
        for (int w = 0; w < AT_WARPS; ++w)
            if (sl[w] != 0.0f) {
                const float f = expf(sm[w] - top);
                sum = fmaf(sa[w][d], f, sum);
                all = fmaf(sl[w], f, all);
            }
        out[i * out_row + h * HD + d] = kv4_from_float<T>(len > 0 ? sum / all : 0.0f);
    }
}

template <typename T>
void launch(const holo_kv4 *c, const Kv4View &view, void *out, const void *q, long long q_row, long long out_row,
            int n_heads, float scale, const int *seqs, int n, cudaStream_t st) {
    const dim3 grid(n_heads, n);
    const int group = n_heads / c->n_kv_heads;
#define HOLO_KV4_SIMPLE(HD)                                                                                      \
    kv4_attn_simple_kernel<T, HD><<<grid, AT_WARPS * 32, 0, st>>>(view, (T *)out, (const T *)q, q_row, out_row, group, \
                                                                  scale, seqs, n)
    switch (c->head_dim) {
    case 64: HOLO_KV4_SIMPLE(64); break;
    case 128: HOLO_KV4_SIMPLE(128); break;
    default: HOLO_KV4_SIMPLE(256); break;
    }
#undef HOLO_KV4_SIMPLE
}

}  // namespace

extern "C" int cuda_kv4_attention(const holo_kv4 *c, int layer, void *out, const void *q, int type, long long q_row,
                                  long long out_row, int n_heads, float scale, const int *seqs, int n) {
    const char *what = "cuda_kv4_attention";
    Kv4View view;
    Kv4Work work;
    cudaStream_t st;
    if (!kv4_begin(c, layer, what, view, st, &work)) return cuda_last_status();
    if (type != HOLO_DT_F32 && type != HOLO_DT_F16 && type != HOLO_DT_BF16) {
        holo_set_status(HOLO_E_UNSUPPORTED, what);
        return HOLO_E_UNSUPPORTED;
    }
    const long long dense = (long long)n_heads * c->head_dim;
    if (q_row == 0) q_row = dense;
    if (out_row == 0) out_row = dense;
    const int size = type == HOLO_DT_F32 ? 4 : 2;
    if (n_heads <= 0 || n_heads % c->n_kv_heads || n < 0 || n > c->max_seqs || q_row < dense || out_row < dense ||
        !(scale >= 0.0f) || (n > 0 && (!out || !q)) || ((uintptr_t)q | (uintptr_t)out) % size) {
        holo_set_status(HOLO_E_ARG, what);
        return HOLO_E_ARG;
    }
    if (n_heads / c->n_kv_heads > KV4_MAX_GROUP || n > 65535) {
        holo_set_status(HOLO_E_UNSUPPORTED, what);
        return HOLO_E_UNSUPPORTED;
    }
    if (n == 0) return HOLO_OK;
    if (scale == 0.0f) scale = 1.0f / sqrtf((float)c->head_dim);
    switch (type) {
    case HOLO_DT_F32: launch<float>(c, view, out, q, q_row, out_row, n_heads, scale, seqs, n, st); break;
    case HOLO_DT_F16: launch<__half>(c, view, out, q, q_row, out_row, n_heads, scale, seqs, n, st); break;
    default: launch<__nv_bfloat16>(c, view, out, q, q_row, out_row, n_heads, scale, seqs, n, st); break;
    }
    return kv4_end(what);
}
