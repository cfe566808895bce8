// kv.cuh — a batch of requests over a paged key/value cache, as the kernels see it (kv_append.cu,
// attn_stream.cu, attn_tile.cu).
#pragma once

#include "stream.cuh"

#include <cuda.h>

namespace tq {

// Status words that a kernel leaves for tq_last_error() (10000 + code) when the batch's device
// arrays say something impossible; what they belong to is skipped, nothing out of range is touched.
constexpr int kStatusBatch = 41;     // token ranges, cached lengths or page numbers out of range
constexpr int kStatusMaxNew = 42;    // a request has more new tokens than the batch's max_new
constexpr int kStatusAdapter = 43;   // an adapter number or rank out of range (lora.cu)

// Whether scratch may be allocated now: not while the stream is captured into a graph.
bool stream_is_capturing();
int gpu_sms();                       // SMs of the device

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
// A bf16 matrix of rows of `cols` values (a multiple of 8, 16-byte aligned), for TMA copies of box_rows rows x 64
// values with the 128-byte swizzle, zeros outside; false if the driver refuses it.
bool tensor_map_2d(CUtensorMap &map, const void *data, int cols, long long rows, int box_rows);
// Whether the memory of two operands has bytes in common.
inline bool overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    return a && b && (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}
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

// ---- the work of an attention call as a line of units ------------------------------------------
// A tile is (request, kv head, ROWS packed query rows: new token x query head of the group); its
// keys are those up to its last row's own, in units of `unit` keys. On the line a tile takes `extra`
// places, for what a tile costs besides its keys, and then one for each unit; the line of all tiles,
// requests outermost, is cut into equal stretches, one per CTA, whatever the lengths.
template <int ROWS>
struct Line {
    const KvArgs &a;
    const int G, unit, extra;
    long long total;             // places of the call
    int ctas;                    // CTAs that have a stretch
    long long base;
    int more;
    long long begin, end;        // this CTA's
    // the tile at hand
    int r, g, m;
    KvRequest q;
    long long at;                // its first place
    int keys, units;

    __device__ Line(const KvArgs &a_, int G_, int unit_, int extra_) : a(a_), G(G_), unit(unit_), extra(extra_) {}
    // The tile's units in this CTA's stretch, [first, last), empty if the stretch ends in the extra
    // places; `from` = the line's place that the stretch enters the tile at.
    __device__ __forceinline__ int first_unit(long long from) const { return (int)max(from - at - extra, 0ll); }
    __device__ __forceinline__ int last_unit() const { return (int)(min((long long)(units + extra), end - at) - extra); }
    __device__ __forceinline__ long long behind() const { return at + extra + units; }

    // A 64-bit division is some hundred instructions: 32 bits wherever the numbers have no more.
    static __device__ __forceinline__ unsigned long long quotient(unsigned long long x, unsigned long long y) {
        return (x | y) >> 32 ? x / y : (unsigned)x / (unsigned)y;
    }
    // n * G stays below 2^31 (checked by the entry point)
    __device__ __forceinline__ int tiles_of(const KvRequest &x) const { return (int)(((unsigned)(x.n * G) + ROWS - 1) / ROWS); }
    __device__ __forceinline__ int tile_keys(const KvRequest &x, int mm) const {
        const int last = min(x.n - 1, (int)(((unsigned)mm * ROWS + ROWS - 1) / (unsigned)G));
        return x.total - x.n + last + 1;
    }
    __device__ __forceinline__ int tile_units(const KvRequest &x, int mm) const {
        return (int)((unsigned)(tile_keys(x, mm) - 1) / (unsigned)unit) + 1;      // a tile has at least one key
    }
    // Places of one kv head of a request. A full tile mm ends at key old + floor((mm ROWS + ROWS - 1) / G), so its
    // units are floor((old G + ROWS - 1 + ROWS mm) / (G unit)) + 1: a sum of floors of a line, by Euclid's steps.
    __device__ long long head_places(const KvRequest &x) const {
        const int tiles = tiles_of(x);
        if (!tiles) return 0;
        long long s = (long long)(extra + 1) * tiles - 1 + tile_units(x, tiles - 1);
        unsigned long long n = tiles - 1, mod = (unsigned long long)G * unit, mul = ROWS,
                           add = (unsigned long long)(x.total - x.n) * G + ROWS - 1;
        while (n) {                                            // s += sum over i < n of floor((mul i + add) / mod)
            const unsigned long long qm = quotient(mul, mod), qa = quotient(add, mod);
            s += (long long)(n * (n - 1) / 2 * qm + n * qa);
            mul -= qm * mod;
            add -= qa * mod;
            const unsigned long long top = mul * n + add;
            n = quotient(top, mod);
            add = top - n * mod;
            const unsigned long long old = mod;
            mod = mul;
            mul = old;
        }
        return s;
    }
    // Start of CTA c's stretch (the first `more` CTAs have base + 1 units, the others base), and the
    // CTA that place u belongs to.
    __device__ __forceinline__ long long start_of(int c) const { return base * c + min(c, more); }
    __device__ __forceinline__ int cta_of(long long u) const {
        const long long cut = (base + 1) * more;
        return u < cut ? (int)quotient(u, base + 1) : more + (int)quotient(u - cut, base);
    }

    // Sum over the threads before this one (block-wide; scan holds THREADS / 32 words), and over all.
    template <int THREADS>
    static __device__ long long scan_before(long long *scan, long long own, long long &all) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        long long sum = own;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += o;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        sum -= own;
        all = 0;
        for (int w = 0; w < THREADS / 32; ++w) {
            const long long v = scan[w];
            if (w < warp) sum += v;
            all += v;
        }
        return sum;
    }
    // Finds this CTA's stretch and its first tile; false if it has none. All THREADS threads of the
    // CTA call it; scan holds THREADS / 32 + 3 words of shared memory.
    template <int THREADS>
    __device__ bool locate(long long *scan, int cta, int grid) {
        constexpr int W = THREADS / 32;
        const int tid = threadIdx.x;
        // the requests' places; those of the first THREADS requests stay at hand
        const long long own0 = tid < a.count ? head_places(kv_request(a, tid)) * a.heads : 0;
        long long mine = own0;
        for (int x = tid + THREADS; x < a.count; x += THREADS) mine += head_places(kv_request(a, x)) * a.heads;
        long long before = scan_before<THREADS>(scan, mine, total);
        ctas = (int)min((long long)grid, total);
        if (cta >= ctas) return false;
        base = quotient(total, ctas);
        more = (int)(total - base * ctas);
        begin = start_of(cta);
        end = start_of(cta + 1);
        // the request that begin lies in, in blocks of THREADS
        long long passed = 0;
        for (int r0 = 0;; r0 += THREADS) {
            const int x = r0 + tid;
            long long own = own0, all = total;
            if (a.count > THREADS) {
                own = r0 == 0 ? own0 : (x < a.count ? head_places(kv_request(a, x)) * a.heads : 0);
                before = scan_before<THREADS>(scan, own, all);
            }
            const long long from = passed + before;
            if (from <= begin && begin < from + own) {
                scan[W] = x;
                scan[W + 1] = from;
                scan[W + 2] = quotient(own, a.heads);
            }
            passed += all;
            if (passed > begin) break;                         // the same in every thread
        }
        __syncthreads();
        r = (int)scan[W];
        at = scan[W + 1];
        q = kv_request(a, r);
        const long long per = scan[W + 2];
        g = (int)quotient(begin - at, per);
        at += per * g;
        // the row tile, in blocks of THREADS
        const int tiles = tiles_of(q);
        passed = at;
        for (int m0 = 0;; m0 += THREADS) {
            const int mm = m0 + tid;
            const int own = mm < tiles ? extra + tile_units(q, mm) : 0;
            long long all;
            const long long from = passed + scan_before<THREADS>(scan, own, all);
            if (from <= begin && begin < from + own) {
                scan[W] = mm;
                scan[W + 1] = from;
            }
            passed += all;
            if (passed > begin) break;
        }
        __syncthreads();
        m = (int)scan[W];
        at = scan[W + 1];
        keys = tile_keys(q, m);
        units = tile_units(q, m);
        return true;
    }
    // The tile behind this one; there is one while behind() < end.
    __device__ __forceinline__ void next() {
        at = behind();
        if (++m == tiles_of(q)) {
            m = 0;
            if (++g == a.heads) {
                g = 0;
                do q = kv_request(a, ++r);
                while (q.n == 0);
            }
        }
        keys = tile_keys(q, m);
        units = tile_units(q, m);
    }
};

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
    const f32x2 minus = pack2(-1.0f, -1.0f);       // x - term as an exact fma, two at a time
    t0 = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    unpack2(fma2(pack2(__uint_as_float(__float_as_uint(x) & 0xffff0000u), bf16_hi(__float_as_uint(y))), minus, pack2(x, y)), x, y);
    t1 = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    unpack2(fma2(pack2(__uint_as_float(__float_as_uint(x) & 0xffff0000u), bf16_hi(__float_as_uint(y))), minus, pack2(x, y)), x, y);
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
