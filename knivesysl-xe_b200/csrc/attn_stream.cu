// attn_stream.cu — attention of few query rows per key/value head over a paged cache (decoding and
// short drafts), and the entry point x_attn_paged that picks between this kernel and attn_tile.cu.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q.k_j) - m),  c = scale * log2(e),  m >= all c (q.k_j)
//
// in one pass over the keys: a warp keeps m, the sum and the weighted values of the keys that it has
// seen, and rescales both when m grows. All queries that read the same key/value head (new tokens x
// query heads of the group) are rows of one mma tile of 16, so the cache is read once.
//
// Each key and value is used for 2 x 16 rows of products at most, so the cache's bytes bound it. The
// work of a call is a line of units of 64 keys over (request, head, row tile); every CTA takes an
// equal stretch of it, whatever the lengths, and its four warps take 16 keys of each unit through
// rings of their own (cp.async, no barrier between warps). A tile that several CTAs share is joined
// by the last of them to finish, in the order of the keys, so results do not depend on timing.
//
// The rule: at most 16 packed rows a head, max_new x group, the same kernel for the whole batch. Decoding
// through the kernel of 128-row tiles instead took 38 us for one request, 159 us for 64 and 187 us for 8
// long e4m3 caches, where this one takes 14, 71 and 78: its ring and its barriers wait for 128 rows of
// products where 16 are wanted. Above 16 rows this one would need a second row tile beside the first (not
// built), or read the cache again for every 16. Measured: 64 requests, bf16, 336 MB of cache: 71 us,
// 4.8 TB/s; 8 long e4m3 caches of dim 256, 171 MB: 78 us, 2.2 TB/s: six query rows in a tile of 16, so most
// products and exponentials are for rows that do not exist, each warp waits on its own chain of conversion,
// product and exponential, and 255 registers leave two warps a scheduler; one request: 13.7 us, latency
// of launch, first bytes and join.
//
// Roundings: the products q.k are exact in the tensor core (bf16 x bf16, or fp16 x fp16 for an e4m3
// cache: e4m3 is exact in fp16, and a query row times a power of two that brings its largest value
// to [2^9, 2^10) loses only what lies 2^-34 below that). Probabilities enter the second product as
// one bf16 term for bf16 outputs (fp16 with an e4m3 cache), and for fp32 outputs as three bf16 terms
// or two fp16 ones, 24 and 22 bits. fp16 ends at 2^-24, so its probabilities are taken 2^15 times as large
// (2^11 in attn_tile.cu), above and below the fraction line: what is lost of one is 2^-40 (2^-36) of the
// row's largest. Without that a key that outweighs the others by 2^16 takes digits from their sum, and one by
// 2^25 all of it. All sums are fp32; for fp32 outputs they leave the tensor core, which
// cuts them off, after every block of 16 keys.
#include "attn.cuh"

#include <algorithm>
#include <math.h>

namespace tq {

namespace {

constexpr int kW = 4;                 // warps of a CTA
constexpr int kKeys = 16;             // keys of a warp's block
constexpr int kUnit = kW * kKeys;     // keys of a unit
constexpr int kRows = 16;             // query rows of a tile
constexpr float kLift = 15.0f;        // of the exponents of fp16 probabilities: the largest is 2^15

template <int D, bool E4M3>
struct Shape {
    static constexpr int kRowBytes = D * (E4M3 ? 1 : 2);
    static constexpr int kBlockBytes = 2 * kKeys * kRowBytes;        // keys and values
    // 24 KB of ring a warp and two CTAs an SM; blocks of 16 KB (D = 256, bf16) three deep, one CTA
    static constexpr int kStages = kBlockBytes >= 16384 ? 3 : 24576 / kBlockBytes;
    static constexpr int kCtas = kBlockBytes >= 16384 ? 1 : 2;
    static constexpr int kRing = kStages * kBlockBytes;
    static constexpr int kSmem = kW * kRing;
    // What a tile costs besides its keys (first loads, the warps' and the CTAs' results joined: some 3 us
    // of a CTA), in units at the rate that all CTAs together read the cache
    static constexpr int kExtra = 65536 / (kW * kBlockBytes) > 1 ? 65536 / (kW * kBlockBytes) : 1;
    // the warps' results of a tile lie over the rings
    static_assert(kW * kRows * D * 4 <= kSmem, "");
};

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same on top of nothing.
template <bool F16>
__device__ __forceinline__ void mma16816_fresh(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

template <int D, bool E4M3, bool OUT_BF16>
__global__ void __launch_bounds__(kW * 32, (Shape<D, E4M3>::kCtas)) attn_stream_kernel(const AttnArgs a) {
    using S = Shape<D, E4M3>;
    constexpr int EB = E4M3 ? 1 : 2;                    // bytes of a cached value
    constexpr int kChunks = S::kRowBytes / 16;          // 16-byte chunks of a row
    constexpr int EPL = 16 / EB;                        // values of a chunk
    constexpr int kGroups = D / (4 * EPL);              // groups of four chunks, one per lane of a quad
    constexpr int kSteps = EPL / 4;                     // k16 steps of a group
    constexpr int NT = D / 8;                           // n8 tiles of the output
    constexpr int kTerms = OUT_BF16 ? 1 : (E4M3 ? 2 : 3);

    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_scan[kW + 3];
    __shared__ int s_join;
    __shared__ float s_m[kW][kRows], s_l[kW][kRows];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.group, cta = blockIdx.x;
    pdl_wait();
    pdl_trigger();

    Line<kRows> line(a.kv, G, kUnit, S::kExtra);
    if (!line.locate<kW * 32>(s_scan, cta, gridDim.x)) return;

    uint8_t *const ring = smem + warp * S::kRing;
    const uint32_t ring_u = smem_u32(ring);
    const int quad = lane & 3, row_a = lane >> 2;      // this thread's tile rows: row_a and row_a + 8

    for (long long u = line.begin;;) {
        // ---- one tile's units [first, last) ------------------------------------------------------
        const KvRequest &req = line.q;
        const int r = line.r, g = line.g, m = line.m, keys = line.keys, units = line.units;
        const int first = line.first_unit(u), last = line.last_unit();
        if (last <= first) break;                      // the stretch ends before the tile's first unit
        const int rows = min(kRows, req.n * G - m * kRows);
        const int blocks = last - first;               // of this warp: one block of 16 keys per unit

        long long next_row;                            // the next block's row numbers, one key per lane
        auto look_up = [&](int b) {                    // rows of block b in the pools; lane & 15 = key
            const int key = (first + b) * kUnit + warp * kKeys + (lane & 15);
            next_row = b < blocks && key < keys ? kv_row(a.kv, r, g, key) : -1;
        };
        auto issue = [&](int b) {                      // block b into its stage; rows from next_row
            if (b < blocks) {
                const uint32_t dst = ring_u + (b % S::kStages) * S::kBlockBytes;
                constexpr int kPerLane = kKeys * kChunks / 32;
#pragma unroll
                for (int i = 0; i < kPerLane; ++i) {
                    const int c = i * 32 + lane, key = c / kChunks, ch = c % kChunks;
                    const long long row = __shfl_sync(0xffffffffu, next_row, key);
                    const size_t off = (size_t)(row < 0 ? 0 : row) * S::kRowBytes + ch * 16;
                    const int swz = (((key & 1) << 2) | ((key >> 1) & 3)) & (kChunks - 1);
                    const uint32_t to = dst + key * S::kRowBytes + ((ch ^ swz) << 4);
                    cp_async16_or_zero(to, a.kv.k + off, row >= 0);
                    cp_async16_or_zero(to + kKeys * S::kRowBytes, a.kv.v + off, row >= 0);
                }
            }
            cp_async_commit();
        };
        look_up(0);
#pragma unroll
        for (int b = 0; b < S::kStages - 1; ++b) {
            issue(b);
            look_up(b + 1);
        }

        // ---- query rows as A fragments: k16 step s of group j holds this lane's values 4s..4s+3 of
        // chunk 4j + quad as its columns {2 quad, +1} and {2 quad + 8, +9}: any order of the summed
        // dimension does as long as both operands have it
        uint32_t qf[kGroups * kSteps][4];
        int limit[2];
        float c_row[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = row_a + 8 * h, rho = m * kRows + i;
            const bool live = i < rows;
            const int tok = rho / G;
            limit[h] = live ? req.total - req.n + tok : -1;
            c_row[h] = a.c;
            const uint16_t *src = a.q + ((size_t)(req.t0 + (live ? tok : 0)) * a.q_heads + g * G + (live ? rho % G : 0)) * D;
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < kGroups; ++j)
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    uint2 v = make_uint2(0, 0);
                    if (live) v = __ldg(reinterpret_cast<const uint2 *>(src + (j * 4 + quad) * EPL + s * 4));
                    qf[j * kSteps + s][h] = v.x;
                    qf[j * kSteps + s][2 + h] = v.y;
                    if constexpr (E4M3) {
                        top = max(top, max(v.x << 16 & 0x7fff0000u, v.x & 0x7fff0000u));
                        top = max(top, max(v.y << 16 & 0x7fff0000u, v.y & 0x7fff0000u));
                    }
                }
            if constexpr (E4M3) {
                // bf16 row -> fp16 row times 2^(9 - exponent of its largest value)
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int ex = min(max((int)(top >> 23) - 127, -100), 127);
                const float up = __uint_as_float((uint32_t)(127 + 9 - ex) << 23);
                c_row[h] = a.c * __uint_as_float((uint32_t)(127 - 9 + ex) << 23);
#pragma unroll
                for (int x = 0; x < kGroups * kSteps; ++x)
#pragma unroll
                    for (int y = h; y < 4; y += 2) {
                        const uint32_t v = qf[x][y];
                        qf[x][y] = pack_f16(bf16_lo(v) * up, bf16_hi(v) * up);
                    }
            }
        }
        const int low = req.total - req.n + m * kRows / G;     // keys up to here are seen by every row

        float o[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[t][x] = 0.0f;
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

        for (int b = 0; b < blocks; ++b) {
            cp_async_wait<S::kStages - 2>();
            __syncwarp();                              // all lanes' copies of block b have landed
            issue(b + S::kStages - 1);                 // its stage was last read in iteration b - 1
            look_up(b + S::kStages);
            const int key0 = (first + b) * kUnit + warp * kKeys;
            if (key0 >= keys) continue;
            const uint32_t kb = ring_u + (b % S::kStages) * S::kBlockBytes;

            // ---- scores of 16 keys: two n8 tiles, each in two sums (a product that adds to the last one's
            // result waits for it)
            float sc[2][4], sc2[2][4];
            uint32_t kline[2];
            int kswz[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int key = t * 8 + row_a;
                sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.0f;
                sc2[t][0] = sc2[t][1] = sc2[t][2] = sc2[t][3] = 0.0f;
                kswz[t] = (((key & 1) << 2) | ((key >> 1) & 3)) & (kChunks - 1);
                kline[t] = kb + key * S::kRowBytes;
            }
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                uint32_t w[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[t][0]), "=r"(w[t][1]), "=r"(w[t][2]), "=r"(w[t][3])
                                 : "r"(kline[t] + (((j * 4 + quad) ^ kswz[t]) << 4)));
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float (&d)[4] = s & 1 ? sc2[t] : sc[t];
                        if constexpr (E4M3)
                            mma16816<true>(d, qf[j * kSteps + s], e4m3_to_f16((uint16_t)w[t][s]), e4m3_to_f16((uint16_t)(w[t][s] >> 16)));
                        else
                            mma16816<false>(d, qf[j * kSteps + s], w[t][2 * s], w[t][2 * s + 1]);
                    }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[t][x] += sc2[t][x];
            // ---- running maximum and probabilities
            const bool cut = key0 + kKeys - 1 > low;
            float p[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v = sc[t][2 * h + x] * c_row[h];
                        if (cut && key0 + t * 8 + quad * 2 + x > limit[h]) v = -INFINITY;
                        p[t][2 * h + x] = v;
                        mx = fmaxf(mx, v);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (mx > top[h]) {
                    const float f = exp2_approx(top[h] - mx);      // 0 the first time
                    top[h] = mx;
                    sum[h] *= f;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        o[t][2 * h] *= f;
                        o[t][2 * h + 1] *= f;
                    }
                }
                const float base = (top[h] == -INFINITY ? 0.0f : top[h]) - (E4M3 ? kLift : 0.0f);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float e = exp2_approx(p[t][2 * h + x] - base);
                        p[t][2 * h + x] = e;
                        sum[h] += e;
                    }
            }
            // ---- the 16 x 16 probabilities as A fragments, split into terms
            uint32_t pf[kTerms][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                // a0: row, keys 2q..; a1: row + 8; a2: row, keys 8 + 2q..; a3: row + 8
                const float lo = p[x >> 1][(x & 1) * 2], hi = p[x >> 1][(x & 1) * 2 + 1];
                if constexpr (kTerms == 3) {
                    split3(lo, hi, pf[0][x], pf[1][x], pf[2][x]);
                } else {
                    pf[0][x] = E4M3 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
                    if constexpr (kTerms == 2) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&pf[0][x]));
                        pf[1][x] = pack_f16(lo - f.x, hi - f.y);
                    }
                }
            }
            // ---- values: ldmatrix.trans gives (2 keys) x (1 b16 unit) per lane
            const int vkey = (lane & 7) + ((lane >> 3) & 1) * 8;
            const int vswz = (((vkey & 1) << 2) | ((vkey >> 1) & 3)) & (kChunks - 1);
            const uint32_t vline = kb + (kKeys + vkey) * S::kRowBytes;
            // A step takes 2 or 4 chunks, four n8 tiles of o. An e4m3 unit holds two neighbouring dims of a key; bytes 0, 2
            // and 1, 3 pair the keys
            constexpr int kPer = E4M3 ? 2 : 1, kStep = 4 / kPer, kOut = 4;       // n8 tiles of a chunk, chunks and tiles of a step
#pragma unroll
            for (int j = 0; j < kChunks; j += kStep) {
                uint32_t w[kStep / 2][4];              // chunk j + i: words 2i (keys 0-7) and 2i + 1 (keys 8-15)
#pragma unroll
                for (int i = 0; i < kStep / 2; ++i) ldmatrix_x4_trans(vline + (((j + 2 * i + (lane >> 4)) ^ vswz) << 4), w[i]);
                uint32_t v[kOut][2];
#pragma unroll
                for (int n = 0; n < kOut; ++n)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int chunk = n / kPer;
                        const uint32_t u16 = w[chunk / 2][chunk % 2 * 2 + y];
                        if constexpr (E4M3) v[n][y] = e4m3_to_f16((uint16_t)__byte_perm(u16, 0, n & 1 ? 0x4431u : 0x4420u));
                        else v[n][y] = u16;
                    }
                if constexpr (kTerms == 1) {
#pragma unroll
                    for (int n = 0; n < kOut; ++n) mma16816<E4M3>(o[j * kPer + n], pf[0], v[n][0], v[n][1]);
                } else {
                    // The tensor core cuts an fp32 sum off instead of rounding it, so a long one falls behind (4e-5 to 9e-5
                    // of itself after 17000 keys): a block's terms, the lower first, have a sum of their own, which an
                    // ordinary addition takes to o (5e-7). 64 decodes: 68 -> 70 us
                    float d[kOut][4];
#pragma unroll
                    for (int n = 0; n < kOut; ++n) mma16816_fresh<E4M3>(d[n], pf[kTerms - 1], v[n][0], v[n][1]);
#pragma unroll
                    for (int k = kTerms - 2; k >= 0; --k)
#pragma unroll
                        for (int n = 0; n < kOut; ++n) mma16816<E4M3>(d[n], pf[k], v[n][0], v[n][1]);
#pragma unroll
                    for (int n = 0; n < kOut; ++n)
#pragma unroll
                        for (int x = 0; x < 4; x += 2) {
                            float (&y)[4] = o[j * kPer + n];
                            unpack2(add2(pack2(y[x], y[x + 1]), pack2(d[n][x], d[n][x + 1])), y[x], y[x + 1]);
                        }
                }
            }
        }
        cp_async_wait<0>();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        }

        // ---- the four warps' results, over the rings: [warp][row][dim]
        __syncthreads();                               // every warp has read its last block
        float *const merged = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = row_a + 8 * h;
            if (row < rows) {
                float *dst = merged + (warp * kRows + row) * D;
                if constexpr (E4M3) {
#pragma unroll
                    for (int t = 0; t < NT; t += 2)    // tiles of even and odd dims of a 16-dim chunk
                        *reinterpret_cast<float4 *>(dst + t * 8 + quad * 4) =
                            make_float4(o[t][2 * h], o[t + 1][2 * h], o[t][2 * h + 1], o[t + 1][2 * h + 1]);
                } else {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        *reinterpret_cast<float2 *>(dst + t * 8 + quad * 2) = make_float2(o[t][2 * h], o[t][2 * h + 1]);
                }
                if (quad == 0) {
                    s_m[warp][row] = top[h];
                    s_l[warp][row] = sum[h];
                }
            }
        }
        __syncthreads();
        const bool whole = first == 0 && last == units;
        // a stretch's first tile goes to part 2 * cta, any later one (the last) to 2 * cta + 1
        float *const part = a.part + (size_t)(2 * cta + (u == line.begin ? 0 : 1)) * kRows * (D + 2);
        auto store = [&](int row, int d, float4 v, float l) {
            const int rho = m * kRows + row, tok = rho / G;
            const float f = l > 0.0f ? __fdiv_rn(a.kv.v_scale, l) : 0.0f;      // no key: a row of zeros
            v.x *= f; v.y *= f; v.z *= f; v.w *= f;
            const size_t to = (size_t)(req.t0 + tok) * a.ldo + (size_t)(g * G + rho % G) * D + d;
            if constexpr (OUT_BF16)
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            else
                *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to) = v;
        };
        for (int x = tid; x < rows * (D / 4); x += kW * 32) {
            const int row = x / (D / 4), d = x % (D / 4) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kW; ++w) M = fmaxf(M, s_m[w][row]);
            const float base = M == -INFINITY ? 0.0f : M;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < kW; ++w) {
                const float f = exp2_approx(s_m[w][row] - base);
                const float4 y = *reinterpret_cast<const float4 *>(merged + (w * kRows + row) * D + d);
                l = fmaf(s_l[w][row], f, l);
                v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
            }
            if (whole) {
                store(row, d, v, l);
            } else {
                *reinterpret_cast<float4 *>(part + row * D + d) = v;
                if (d == 0) {
                    part[kRows * D + row] = M;
                    part[kRows * D + kRows + row] = l;
                }
            }
        }
        if (!whole) {
            const int c0 = line.cta_of(line.at + S::kExtra), c1 = line.cta_of(line.behind() - 1);    // share the tile
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int n = atomicAdd(a.arrived + c0, 1);
                s_join = n == c1 - c0;
                if (s_join) a.arrived[c0] = 0;         // ready for the next call
            }
            __syncthreads();
            if (s_join) {
                __threadfence();
                const int slot0 = line.start_of(c0) >= line.at ? 2 * c0 : 2 * c0 + 1;
                for (int x = tid; x < rows * (D / 4); x += kW * 32) {
                    const int row = x / (D / 4), d = x % (D / 4) * 4;
                    float M = -INFINITY, l = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int c = c0; c <= c1; ++c) {
                        const float *src = a.part + (size_t)(c == c0 ? slot0 : 2 * c) * kRows * (D + 2);
                        const float mc = __ldcg(src + kRows * D + row), lc = __ldcg(src + kRows * D + kRows + row);
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(src + row * D + d));
                        const float Mn = fmaxf(M, mc), base = Mn == -INFINITY ? 0.0f : Mn;
                        const float f = exp2_approx(M - base), fc = exp2_approx(mc - base);
                        M = Mn;
                        l = fmaf(lc, fc, l * f);
                        v.x = fmaf(y.x, fc, v.x * f); v.y = fmaf(y.y, fc, v.y * f);
                        v.z = fmaf(y.z, fc, v.z * f); v.w = fmaf(y.w, fc, v.w * f);
                    }
                    store(row, d, v, l);
                }
            }
        }
        __syncthreads();                               // the rings are free again

        u = line.behind();
        if (u >= line.end) break;
        line.next();
    }
}

struct AttnScratch {
    float *part = nullptr;
    int *arrived = nullptr;
};
AttnScratch g_attn;

// The same for every call, whatever its sizes: parts of two tiles for each CTA of either kernel.
int attn_scratch(int sms) {
    if (g_attn.part) return 0;
    if (stream_is_capturing()) return -40;
    const size_t stream_floats = (size_t)2 * 2 * sms * kRows * (256 + 2);
    g_attn.part = static_cast<float *>(tq_dev_alloc(std::max(stream_floats, attn_tile_part_floats(sms)) * sizeof(float), "attn.part"));
    g_attn.arrived = static_cast<int *>(tq_dev_alloc((size_t)2 * sms * sizeof(int), "attn.arrived"));
    TQ_CHECK(cudaMemsetAsync(g_attn.arrived, 0, (size_t)2 * sms * sizeof(int), stream()));
    return 0;
}

template <int D, bool E4M3, bool OUT_BF16>
void launch_stream(const AttnArgs &a) {
    using S = Shape<D, E4M3>;
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(attn_stream_kernel<D, E4M3, OUT_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        set = true;
    }
    launch_pdl(attn_stream_kernel<D, E4M3, OUT_BF16>, dim3(gpu_sms() * S::kCtas), dim3(kW * 32), (size_t)S::kSmem, a);
    TQ_LAUNCH_CHECK("attn_stream_kernel");
}
template <int D>
void launch_stream(const AttnArgs &a, bool e4m3) {
    if (e4m3) a.out_bf16 ? launch_stream<D, true, true>(a) : launch_stream<D, true, false>(a);
    else a.out_bf16 ? launch_stream<D, false, true>(a) : launch_stream<D, false, false>(a);
}

}  // namespace
}  // namespace tq

int x_attn_paged(const tq_kv_cache_t *cache, const tq_kv_batch_t *batch, const uint16_t *d_q, int q_heads, float scale,
                 void *d_out, size_t ldo, int out_bf16) {
    using namespace tq;
    AttnArgs a{};
    if (const int rc = kv_args(cache, batch, a.kv)) return rc;
    const int D = a.kv.dim;
    if (q_heads <= 0 || !(fabsf(scale) < INFINITY) || (out_bf16 != 0 && out_bf16 != 1)) return -2;
    a.c = scale * a.kv.k_scale * 1.4426950408889634f;
    if (!(fabsf(a.c) < INFINITY)) return -2;
    if (q_heads % a.kv.heads || q_heads > 65535) return -3;
    if (!a.kv.count || !a.kv.tokens || !a.kv.max_new) return 0;
    if (!d_q || !d_out || ldo < (size_t)q_heads * D) return -2;
    // packed rows (new tokens x group) are counted in 32 bits
    if ((long long)a.kv.tokens * q_heads > 0x7fffff00ll) return -3;
    if (!aligned16(d_q) || !aligned16(d_out) || ldo % (out_bf16 ? 8 : 4)) return -4;
    // A tile's rows are written after all that read its queries have done so: in place the two may be the same rows
    const size_t width = (size_t)q_heads * D, q_bytes = a.kv.tokens * width * 2;
    const size_t out_bytes = ((a.kv.tokens - 1) * ldo + width) * (out_bf16 ? 2 : 4);
    if (overlap(d_out, out_bytes, d_q, q_bytes) && !(d_out == d_q && out_bf16 && ldo == width)) return -2;
    if (const int rc = attn_scratch(gpu_sms())) return rc;
    if (!device_status_ready()) return -40;
    a.kv.status = device_status_word();
    a.q = d_q;
    a.out = d_out;
    a.ldo = ldo;
    a.q_heads = q_heads;
    a.group = q_heads / a.kv.heads;
    a.out_bf16 = out_bf16;
    a.part = g_attn.part;
    a.arrived = g_attn.arrived;
    a.limit_ns = wait_limit_ns();
    const bool e4m3 = cache->e4m3 != 0;
    if ((long long)a.kv.max_new * a.group > kRows) {
        launch_attn_tile(a, e4m3, gpu_sms());
        return 0;
    }
    if (D == 64) launch_stream<64>(a, e4m3);
    else if (D == 128) launch_stream<128>(a, e4m3);
    else launch_stream<256>(a, e4m3);
    return 0;
}
