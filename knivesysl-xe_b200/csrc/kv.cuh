// kv.cuh — a batch of requests over a paged key/value cache, as the kernels see it (kv_append.cu,
// attn_stream.cu, attn_tile.cu).
#pragma once

#include "stream.cuh"

namespace tq {

// Status words that a kernel leaves for tq_last_error() (10000 + code) when the batch's device
// arrays say something impossible; what they belong to is skipped, nothing out of range is touched.
constexpr int kStatusBatch = 41;     // token ranges, cached lengths or page numbers out of range
constexpr int kStatusMaxNew = 42;    // a request has more new tokens than the batch's max_new
constexpr int kStatusAdapter = 43;   // an adapter number or rank out of range (lora.cu)

// Whether scratch may be allocated now: not while the stream is captured into a graph.
bool stream_is_capturing();

struct KvArgs {
    uint8_t *k, *v;              // [pages][heads][page_size][dim]
    int pages, page_size, heads, dim;
    float k_scale, v_scale;      // 1 for bf16
    const int *start, *kv_len, *page;
    int count, tokens, max_new, max_pages;
    int *status;
};
// Checks the two records; 0 and the kernels' view of them, else the entry points' return code.
int kv_args(const tq_kv_cache_t *cache, const tq_kv_batch_t *batch, KvArgs &a);
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

#ifdef __CUDACC__

// New tokens [t0, t0 + n) of the batch's rows, at positions total - n .. total - 1.
struct KvRequest {
    int t0, n, total;
};
__device__ __forceinline__ KvRequest kv_request(const KvArgs &a, int r) {
    const int t0 = __ldg(a.start + r), t1 = __ldg(a.start + r + 1), total = __ldg(a.kv_len + r);
    const long long room = (long long)a.max_pages * a.page_size;
    int bad = 0;
    if (t0 < 0 || t1 < t0 || t1 > a.tokens || total < 0 || total > room || (long long)t1 - t0 > total) bad = kStatusBatch;
    else if (t1 - t0 > a.max_new) bad = kStatusMaxNew;
    if (bad) {
        atomicCAS(a.status, 0, bad);
        return {0, 0, 0};
    }
    return {t0, t1 - t0, total};
}

// Row (of dim values) of position p of request r in the pools for kv head g; -1 where the page
// table names no page of the pool.
__device__ __forceinline__ long long kv_row(const KvArgs &a, int r, int g, int p) {
    const int page = __ldg(a.page + (size_t)r * a.max_pages + p / a.page_size);
    if (page < 0 || page >= a.pages) {
        atomicCAS(a.status, 0, kStatusBatch);
        return -1;
    }
    return ((long long)page * a.heads + g) * a.page_size + p % a.page_size;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 values rounded to nearest, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// Three bf16 terms of each of a pair of fp32 values, cut off instead of rounded: 8 bits each, their sum
// is the value (of a value that is not finite, NaN).
__device__ __forceinline__ void split3(float x, float y, uint32_t &t0, uint32_t &t1, uint32_t &t2) {
    t0 = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= bf16_lo(t0);
    y -= bf16_hi(t0);
    t1 = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= bf16_lo(t1);
    y -= bf16_hi(t1);
    t2 = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
// Two e4m3 values (low byte first) as fp16, exactly.
__device__ __forceinline__ uint32_t e4m3_to_f16(uint16_t v) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(v));
    return d;
}
// Rounded to nearest, beyond +-448 to +-448.
__device__ __forceinline__ uint16_t pack_e4m3(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}

#endif  // __CUDACC__

}  // namespace tq
