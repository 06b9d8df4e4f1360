// kv4.cuh -- the paged 4-bit KV cache: block layout (holo_b200.h), addressing,
// row types, and the workspace shared by kv4_cache.cu (rows in and out),
// kv4_attn.cu (single-token attention) and kv4_pages.cu (allocation, forks,
// moves).
#pragma once
#include "holo_common.cuh"

#include <cuda_bf16.h>

constexpr int KV4_BLOCK = 16;          // positions a block
constexpr int KV4_GROUP = 32;          // values a scale
constexpr int KV4_HEADS = 8;           // query heads of one KV head that one work item of the attention takes (MMA N)
constexpr int KV4_MAX_GROUP = 16;      // query heads a KV head
constexpr int KV4_MAX_CTAS = 1024;     // CTAs of the attention (two partial results each)

// byte offsets inside a block of head size hd (all multiples of 16)
__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 18 * hd; }
__host__ __device__ constexpr int kv4_off_v(int hd) { return 8 * hd; }
__host__ __device__ constexpr int kv4_off_dk(int hd) { return 16 * hd; }
__host__ __device__ constexpr int kv4_off_dv(int hd) { return 17 * hd; }
// the halfword with values 32 b + 4 g .. + 3 of a position: of its key codes
// (half of the word (quarter g / 2, group b)) and of its value codes
__host__ __device__ constexpr int kv4_k_half(int hd, int pos, int g, int b) {
    return pos * (hd / 2) + ((g >> 1) * (hd / 32) + b) * 4 + (g & 1) * 2;
}
__host__ __device__ constexpr int kv4_v_half(int hd, int pos, int g, int b) {
    return (((((g >> 1) * 8 + (pos >> 1)) * 2 + (g & 1)) * 2 + (pos & 1)) * (hd / 32) + b) * 2;
}

// what the kernels need of a holo_kv4, by value
struct Kv4View {
    uint8_t *pool;                     // of the layer
    int *tables, *lens, *refs;
    int n_kv, page_tokens, page_blocks, n_pages, max_seqs, max_pages;
    int *status;
};

// sections of the workspace: the attention's counters (zero between calls),
// the page operators' lists, the attention's partial results
struct Kv4Work {
    int *counters;                     // [max_seqs * n_kv * KV4_MAX_GROUP / KV4_HEADS]
    int *plan;                         // [16 + 3 * n_pages + 2 * max_seqs]
    float *partial;                    // [KV4_MAX_CTAS][2][KV4_HEADS][hd + 2]
};

bool kv4_shape_ok(const holo_kv4 *c);
// Checks c (and, for what >= 0, the layer), and takes its stream and, with
// `work`, its workspace; false with the status set.
bool kv4_begin(const holo_kv4 *c, int layer, const char *what, Kv4View &view, cudaStream_t &st, Kv4Work *work);
// the status of a call: of the launch before it
int kv4_end(const char *what);

#ifdef __CUDACC__

__device__ __forceinline__ void kv4_report(int *status, int code) { atomicCAS(status, 0, code); }

__device__ __forceinline__ uint8_t *kv4_block(const Kv4View &c, int hd, int page, int kvh, int block) {
    return c.pool + (((size_t)page * c.n_kv + kvh) * c.page_blocks + block) * kv4_block_bytes(hd);
}

template <typename T> __device__ __forceinline__ float kv4_to_float(T x);
template <> __device__ __forceinline__ float kv4_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float kv4_to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float kv4_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T kv4_from_float(float x);
template <> __device__ __forceinline__ float kv4_from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half kv4_from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 kv4_from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

#endif  // __CUDACC__
