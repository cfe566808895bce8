// attn_tile.cu — attention of chunks of new tokens over a paged cache on tcgen05 (x_attn_paged).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m)
//
// A tile is 128 packed query rows (new token x query head) of one key/value head; a CTA carries two
// of them (one for dim 256), each with its own scores S and sums O in tensor memory, so that the
// tensor core multiplies for one while the other's probabilities are computed. Roles:
//   softmax  one warpgroup per tile, a thread per row: its queries into shared memory, then per block
//            of keys S -> running maximum -> P, written over S as the next product's A operand
//   load     four warps: the blocks of keys and values, page by page, into a ring in shared memory
//            (cp.async; an e4m3 cache passes through registers, where it becomes fp16)
//   mma      one warp: S = Q K^T and O += P V, and the barriers that free ring and rows
// O is rescaled only when a row's maximum grows by more than 2^8: until then probabilities are up to
// 2^8 instead of 1, which costs no precision, and the rescaling pass over O hardly ever runs.
//
// Two products of 128 x 128 x dim and 128 x 128 exponentials take about the same time on an SM
// (1024 clocks at dim 128), which bounds this kernel; the cache is read once per 256 rows.
//
// Work is cut into equal stretches of key blocks, one per SM (Line, kv.cuh): a causal batch of any
// lengths loads all SMs alike. A tile cut between CTAs leaves (m, sum, O) of each part in global
// memory, and a second, small kernel joins them in the order of the keys.
//
// Roundings: as in attn_stream.cu.
#include "attn.cuh"
#include "tc.cuh"

#include <algorithm>
#include <type_traits>

namespace tq {

namespace {

constexpr int kRowsTile = 128;
constexpr int kLoadWarps = 4;

template <int D, bool E4M3, int TERMS>
struct TileShape {
    static constexpr int kTiles = D <= 128 ? 2 : 1;                 // row tiles of a CTA
    static constexpr int kRows = kRowsTile * kTiles;
    // keys of a block. More terms of P need tensor memory, dim 256 shared memory: 64 then
    static constexpr int kKeys = TERMS == 1 && D <= 128 ? 128 : 64;
    static constexpr int kBlock = kKeys * D * 2;                    // bytes of keys, or of values
    static constexpr int kSlots = 131072 / kBlock > 8 ? 8 : 131072 / kBlock;
    static constexpr int kQ = kRowsTile * D * 2;                    // bytes of a tile's queries
    static constexpr int kSmem = kTiles * kQ + kSlots * kBlock + 1024;
    static constexpr int kSoftmax = kTiles * 128;                   // threads
    static constexpr int kThreads = kSoftmax + kLoadWarps * 32 + 32;
};

// 128-byte swizzle: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7), groups of 8 rows 1024
// bytes apart (SBO). K-major operands step 32 bytes per k16; MN-major ones (values: the summed
// dimension runs over rows) have their next 64 columns LBO bytes further on.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// kind::f16: D = f32, A and B fp16 or bf16; B may be MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool bf16, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
#define TQ_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define TQ_RW8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
// 32 columns of this thread's lane; the registers are valid behind tmem_wait32 on the same array.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : TQ_R8(v, 0), TQ_R8(v, 8), TQ_R8(v, 16), TQ_R8(v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TQ_RW8(v, 0), TQ_RW8(v, 8), TQ_RW8(v, 16), TQ_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void cp_async16_zero_fill(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A wait of this kernel, by a whole warp: bounded, and given up at once when another wait of the CTA was.
struct Waits {
    volatile int *gave_up;
    int *status;
    unsigned long long limit_ns;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
        if (mbar_test_wait_warp(bar, parity)) return true;
        bool ok = false;
        if (!*gave_up) {
            ok = mbar_wait_slow(bar, parity, status, 24, limit_ns);
            if (!ok) *gave_up = 1;
        }
        return __all_sync(0xffffffffu, ok);
    }
};

// The parts of a tile that a CTA started and others finished, for the join kernel: rows of the
// output and the CTAs that have parts. count = 0: none.
struct JoinTile {
    int t0, n, g, m;             // first token, new tokens, kv head, row block
    int c0, c1, slot0;
    int count;
};

template <int D, bool E4M3, int TERMS>
__global__ void __launch_bounds__((TileShape<D, E4M3, TERMS>::kThreads), 1) attn_tile_kernel(const AttnArgs a, JoinTile *joins) {
    using S = TileShape<D, E4M3, TERMS>;
    constexpr int kT = S::kTiles, kN = S::kKeys;
    constexpr bool OUT_BF16 = TERMS == 1;
    constexpr uint32_t kSlotCol = 256;                 // tensor memory: O tiles, then two slots of 128 columns (S, P)
    constexpr uint32_t kQkDesc = idesc_f16(128, kN, !E4M3, false), kPvDesc = idesc_f16(128, D, !E4M3, true);

    extern __shared__ uint8_t smem_raw[];
    __shared__ long long s_scan[S::kThreads / 32 + 3];
    __shared__ __align__(8) uint64_t s_bar[2 * S::kSlots + 2 * 2 + 2 * kT + 1];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    const int G = a.group;
    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_smem = base, ring = base + kT * S::kQ;
    const uint32_t bars = smem_u32(s_bar);
    auto full = [&](int i) { return bars + 8 * i; };                        // ring slot holds a block
    auto empty = [&](int i) { return bars + 8 * (S::kSlots + i); };         // and may be written again
    auto s_full = [&](int i) { return bars + 8 * (2 * S::kSlots + i); };    // slot i holds scores
    auto p_full = [&](int i) { return bars + 8 * (2 * S::kSlots + 2 + i); };
    auto q_full = [&](int i) { return bars + 8 * (2 * S::kSlots + 4 + i); };
    auto o_done = [&](int i) { return bars + 8 * (2 * S::kSlots + 4 + kT + i); };   // a P V product of tile i is complete
    const uint32_t drained = bars + 8 * (2 * S::kSlots + 4 + 2 * kT);       // all products and their arrivals are done

    if (tid == 0) {
        mbar_init(drained, 1);
        for (int i = 0; i < S::kSlots; ++i) {
            mbar_init(full(i), kLoadWarps);
            mbar_init(empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), 4);
        }
        for (int i = 0; i < kT; ++i) {
            mbar_init(q_full(i), 4);
            mbar_init(o_done(i), 1);
        }
        mbar_init_fence();
        s_gave_up = 0;
    }
    pdl_wait();
    pdl_trigger();
    Line<S::kRows> line(a.kv, G, kN, 2);
    const bool work = line.template locate<S::kThreads>(s_scan, cta, gridDim.x);
    if (tid == 0) joins[cta].count = 0;
    if (!work) return;
    constexpr int kMmaWarp = S::kSoftmax / 32 + kLoadWarps;
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Waits wait{&s_gave_up, a.kv.status, a.limit_ns};

    // Of tile t in the units [first, last) of the block of rows at hand: rows, and the end of its own units.
    auto tile_rows = [&](int t) {
        const long long left = (long long)line.q.n * G - (long long)line.m * S::kRows - t * kRowsTile;
        return (int)min((long long)kRowsTile, max(left, 0ll));
    };
    auto tile_end = [&](int t, int last) {
        const int rows = tile_rows(t);
        if (!rows) return 0;
        const int tok = (line.m * S::kRows + t * kRowsTile + rows - 1) / G;
        return min(last, (line.q.total - line.q.n + tok) / kN + 1);
    };

    if (warp < S::kSoftmax / 32) {
        // ================================ softmax ================================================
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lane_col = tmem + ((uint32_t)(warp & 3) << 21);
        const uint32_t o_col = lane_col + t * D;
        uint32_t s_phase = 0, o_count = 0;               // a bit per slot; products of this tile
        bool alive = true;
        for (long long u = line.begin; alive;) {
            const KvRequest req = line.q;
            const int first = line.first_unit(u), last = line.last_unit();
            if (last <= first) break;
            const int end = tile_end(t, last), rows = tile_rows(t);
            const int rho = line.m * S::kRows + t * kRowsTile + row, tok = rho / G;
            const bool live = row < rows;
            const int limit = live ? req.total - req.n + tok : -1;
            const int low = req.total - req.n + (line.m * S::kRows + t * kRowsTile) / G;   // seen by all rows
            float c = fabsf(a.c), m = -INFINITY, l = 0.0f;
            if (first < end) {
                // ---- the warp's 32 rows of queries, turned by the sign of the scale, whole rows per load
                const uint32_t flip = a.c < 0.0f ? 0x80008000u : 0u, keep = a.c != 0.0f ? 0xffffffffu : 0u;
                const long long mine = live ? ((long long)(req.t0 + tok) * a.q_heads + line.g * G + rho % G) * D : -1;
                const uint32_t q_tile = q_smem + t * S::kQ;
                constexpr int kQChunks = D / 8;            // 16-byte chunks of a row
                uint4 v[8];
#pragma unroll
                for (int x0 = 0; x0 < kQChunks; x0 += 8) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int i = (x0 + x) * 32 + lane;
                        const long long from = __shfl_sync(0xffffffffu, mine, i / kQChunks);
                        v[x] = from >= 0 ? __ldg(reinterpret_cast<const uint4 *>(a.q + from) + i % kQChunks) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int i = (x0 + x) * 32 + lane, r = (warp & 3) * 32 + i / kQChunks, ch = i % kQChunks;
                        st_shared16(q_tile + (ch >> 3) * (kRowsTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                                    make_uint4((v[x].x ^ flip) & keep, (v[x].y ^ flip) & keep, (v[x].z ^ flip) & keep,
                                               (v[x].w ^ flip) & keep));
                    }
                }
                if constexpr (E4M3) {
                    // own row: to fp16, times the power of two that takes its largest value to [2^9, 2^10)
                    __syncwarp();
                    auto place = [&](int ch) { return q_tile + (ch >> 3) * (kRowsTile * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4); };
                    uint32_t top = 0;
#pragma unroll 8
                    for (int ch = 0; ch < kQChunks; ++ch) {
                        const uint4 w = ld_shared16(place(ch));
                        top = max(max(top, max(w.x << 16 & 0x7fff0000u, w.x & 0x7fff0000u)), max(w.y << 16 & 0x7fff0000u, w.y & 0x7fff0000u));
                        top = max(max(top, max(w.z << 16 & 0x7fff0000u, w.z & 0x7fff0000u)), max(w.w << 16 & 0x7fff0000u, w.w & 0x7fff0000u));
                    }
                    const int ex = min(max((int)(top >> 23) - 127, -100), 127);
                    const float by = __uint_as_float((uint32_t)(127 + 9 - ex) << 23);
                    c *= __uint_as_float((uint32_t)(127 - 9 + ex) << 23);
#pragma unroll 8
                    for (int ch = 0; ch < kQChunks; ++ch) {
                        const uint4 w = ld_shared16(place(ch));
                        st_shared16(place(ch), make_uint4(pack_f16(bf16_lo(w.x) * by, bf16_hi(w.x) * by), pack_f16(bf16_lo(w.y) * by, bf16_hi(w.y) * by),
                                                          pack_f16(bf16_lo(w.z) * by, bf16_hi(w.z) * by), pack_f16(bf16_lo(w.w) * by, bf16_hi(w.w) * by)));
                    }
                }
                if (!(c > 0.0f)) c = 1.17549435e-38f;      // scores of no size: any factor above 0
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full(t));

                for (int j = first; j < end; ++j) {
                    const int slot = kT == 2 ? t : (j - first) & 1;
                    const uint32_t s_col = lane_col + kSlotCol + slot * 128;
                    if (!wait(s_full(slot), s_phase >> slot & 1)) { alive = false; break; }
                    s_phase ^= 1u << slot;
                    tc_fence_after();
                    const int key0 = j * kN;
                    const bool cut = key0 + kN - 1 > low;
                    // ---- maximum of the block, the next columns' load under it
                    float mx = -INFINITY;
                    auto largest = [&](auto is_cut) {
                        uint32_t v[2][32];
                        tmem_ld32(s_col, v[0]);
#pragma unroll
                        for (int x = 0; x < kN; x += 32) {
                            uint32_t (&w)[32] = v[x / 32 & 1];
                            tmem_wait32(w);
                            if (x + 32 < kN) tmem_ld32(s_col + x + 32, v[x / 32 & 1 ^ 1]);
                            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                            for (int y = 0; y < 32; y += 2) {
                                if constexpr (decltype(is_cut)::value) {
                                    if (key0 + x + y <= limit) m0 = fmaxf(m0, __uint_as_float(w[y]));
                                    if (key0 + x + y + 1 <= limit) m1 = fmaxf(m1, __uint_as_float(w[y + 1]));
                                } else {
                                    m0 = fmaxf(m0, __uint_as_float(w[y]));
                                    m1 = fmaxf(m1, __uint_as_float(w[y + 1]));
                                }
                            }
                            mx = fmaxf(mx, fmaxf(m0, m1));
                        }
                    };
                    if (cut) largest(std::true_type());
                    else largest(std::false_type());
                    mx *= c;
                    const bool grows = mx > m + 8.0f;
                    if (j > first && __any_sync(0xffffffffu, grows)) {
                        // the product of block j - 1 must be in O
                        if (!wait(o_done(t), (o_count - 1) & 1)) { alive = false; break; }
                        tc_fence_after();
                        const float f = grows ? exp2_approx(m - mx) : 1.0f;
                        l *= f;
#pragma unroll
                        for (int x = 0; x < D; x += 32) {
                            uint32_t v[32];
                            tmem_ld32(o_col + x, v);
                            tmem_wait32(v);
#pragma unroll
                            for (int y = 0; y < 32; ++y) v[y] = __float_as_uint(__uint_as_float(v[y]) * f);
                            uint32_t w[16];
#pragma unroll
                            for (int y = 0; y < 16; ++y) w[y] = v[y];
                            tmem_st16(o_col + x, w);
#pragma unroll
                            for (int y = 0; y < 16; ++y) w[y] = v[16 + y];
                            tmem_st16(o_col + x + 16, w);
                        }
                    }
                    if (grows) m = mx;
                    const float off = m == -INFINITY ? 0.0f : -m;
                    // ---- probabilities, over the scores already read
                    f32x2 sum = pack2(0.0f, 0.0f);
                    const f32x2 c2 = pack2(c, c), off2 = pack2(off, off);
                    auto weights = [&](auto is_cut) {
                        uint32_t v[2][32];
                        tmem_ld32(s_col, v[0]);
#pragma unroll
                        for (int x = 0; x < kN; x += 32) {
                            uint32_t (&sc)[32] = v[x / 32 & 1];
                            tmem_wait32(sc);
                            if (x + 32 < kN) tmem_ld32(s_col + x + 32, v[x / 32 & 1 ^ 1]);
                            uint32_t w[TERMS][16];
#pragma unroll
                            for (int y = 0; y < 32; y += 2) {
                                float p0, p1;
                                unpack2(fma2(pack2(__uint_as_float(sc[y]), __uint_as_float(sc[y + 1])), c2, off2), p0, p1);
                                p0 = exp2_approx(p0);
                                p1 = exp2_approx(p1);
                                if constexpr (decltype(is_cut)::value) {
                                    if (key0 + x + y > limit) p0 = 0.0f;
                                    if (key0 + x + y + 1 > limit) p1 = 0.0f;
                                }
                                sum = add2(sum, pack2(p0, p1));
                                if constexpr (TERMS == 3) {
                                    split3(p0, p1, w[0][y / 2], w[1][y / 2], w[2][y / 2]);
                                } else {
                                    w[0][y / 2] = E4M3 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
                                    if constexpr (TERMS == 2) {
                                        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[0][y / 2]));
                                        w[1][y / 2] = pack_f16(p0 - f.x, p1 - f.y);
                                    }
                                }
                            }
                            tmem_st16(s_col + x / 2, w[0]);
                            if constexpr (TERMS >= 2) tmem_st16(s_col + 64 + x / 2, w[1]);
                            if constexpr (TERMS == 3) tmem_st16(s_col + 96 + x / 2, w[2]);
                        }
                    };
                    if (cut) weights(std::true_type());
                    else weights(std::false_type());
                    float l0, l1;
                    unpack2(sum, l0, l1);
                    l += l0 + l1;
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(slot));
                    ++o_count;
                }
                if (!alive || !wait(o_done(t), (o_count - 1) & 1)) break;
                tc_fence_after();
            }
            // ---- the tile's rows, or this CTA's part of them
            const bool whole = first == 0 && last == line.units;
            if (whole) {
                const float f = l > 0.0f ? __fdiv_rn(a.kv.v_scale, l) : (l == l ? 0.0f : l);
                const size_t to = (size_t)(req.t0 + tok) * a.ldo + (size_t)(line.g * G + rho % G) * D;
                if (first < end)
#pragma unroll
                    for (int x = 0; x < D; x += 32) {
                        uint32_t v[32];
                        tmem_ld32(o_col + x, v);
                        tmem_wait32(v);
                        if (!live) {
                        } else if constexpr (OUT_BF16) {
                            uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to + x);
#pragma unroll
                            for (int y = 0; y < 32; y += 8) {
                                uint32_t w[4];
#pragma unroll
                                for (int z = 0; z < 4; ++z)
                                    w[z] = pack_bf16(__uint_as_float(v[y + 2 * z]) * f, __uint_as_float(v[y + 2 * z + 1]) * f);
                                dst[y / 8] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
                            float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to + x);
#pragma unroll
                            for (int y = 0; y < 32; y += 4)
                                dst[y / 4] = make_float4(__uint_as_float(v[y]) * f, __uint_as_float(v[y + 1]) * f,
                                                         __uint_as_float(v[y + 2]) * f, __uint_as_float(v[y + 3]) * f);
                        }
                        __syncwarp();
                    }
            } else {
                // [dim][row]: neighbouring threads write neighbouring words
                const int slot = 2 * cta + (u == line.begin ? 0 : 1);
                float *part = a.part + (size_t)(slot * kT + t) * (D + 2) * kRowsTile + row;
                if (first < end)
#pragma unroll
                    for (int x = 0; x < D; x += 32) {
                        uint32_t v[32];
                        tmem_ld32(o_col + x, v);
                        tmem_wait32(v);
#pragma unroll
                        for (int y = 0; y < 32; ++y) part[(x + y) * kRowsTile] = __uint_as_float(v[y]);
                    }
                part[D * kRowsTile] = m;
                part[(D + 1) * kRowsTile] = l;
            }
            tc_fence_before();
            if (tid == 0 && first == 0 && last < line.units)      // the tile starts here and goes on: its parts
                joins[cta] = JoinTile{req.t0, req.n, line.g, line.m, cta, line.cta_of(line.behind() - 1),
                                      2 * cta + (u == line.begin ? 0 : 1), 1};
            u = line.behind();
            if (u >= line.end) break;
            line.next();
        }
    } else if (warp < kMmaWarp) {
        // ================================ load ===================================================
        constexpr int kKeysW = kN / kLoadWarps;            // keys of a warp
        constexpr int kChunks = (E4M3 ? D : 2 * D) / 16;   // of a cached row
        constexpr int kLoads = kKeysW * kChunks / 32;
        const int w = warp - S::kSoftmax / 32;
        int at = 0;                                        // blocks so far; slot at % kSlots
        int told = 0;                                      // of them, handed over
        bool alive = true;
        auto hand_over = [&](int upto) {
            fence_proxy_async_smem();
            __syncwarp();
            for (; told < upto; ++told)
                if (lane == 0) mbar_arrive(full(told % S::kSlots));
        };
        auto wait_empty = [&]() {
            if (at < S::kSlots) return true;
            const uint32_t bar = empty(at % S::kSlots), parity = ((at / S::kSlots) - 1) & 1;
            if constexpr (!E4M3) {
                if (!mbar_test_wait_warp(bar, parity)) {   // before a wait, what has been started is finished and handed over
                    cp_async_wait<0>();
                    hand_over(at);
                }
            }
            return wait(bar, parity);
        };
        for (long long u = line.begin; alive;) {
            const int first = line.first_unit(u), last = line.last_unit();
            if (last <= first) break;
            auto look_up = [&](int j) {
                const int key = j * kN + w * kKeysW + (lane % kKeysW);
                return j < last && key < line.keys ? kv_row(a.kv, line.r, line.g, key) : -1ll;
            };
            long long row = look_up(first);
            if constexpr (E4M3) {
                uint4 held[kLoads];
                auto load = [&](const uint8_t *pool) {
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int x = i * 32 + lane;
                        const long long r = __shfl_sync(0xffffffffu, row, x / kChunks);
                        held[i] = r >= 0 ? __ldg(reinterpret_cast<const uint4 *>(pool + (size_t)r * D + (x % kChunks) * 16))
                                         : make_uint4(0, 0, 0, 0);
                    }
                };
                auto store = [&]() {                       // chunk of 16 values -> two of 8 fp16 values
                    const uint32_t dst = ring + (at % S::kSlots) * S::kBlock;
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int x = i * 32 + lane, key = w * kKeysW + x / kChunks, ch = x % kChunks * 2;
                        const uint32_t to = dst + (ch >> 3) * (kN * 128) + key * 128;
                        const uint32_t v[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
                        uint32_t f[8];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            f[2 * y] = e4m3_to_f16((uint16_t)v[y]);
                            f[2 * y + 1] = e4m3_to_f16((uint16_t)(v[y] >> 16));
                        }
                        st_shared16(to + (((ch & 7) ^ (key & 7)) << 4), make_uint4(f[0], f[1], f[2], f[3]));
                        st_shared16(to + ((((ch & 7) + 1) ^ (key & 7)) << 4), make_uint4(f[4], f[5], f[6], f[7]));
                    }
                };
                load(a.kv.k);
                for (int j = first; j < last; ++j) {
                    if (!wait_empty()) { alive = false; break; }
                    store();
                    hand_over(++at);
                    load(a.kv.v);
                    row = look_up(j + 1);
                    if (!wait_empty()) { alive = false; break; }
                    store();
                    hand_over(++at);
                    load(a.kv.k);
                }
            } else {
                for (int j = first; j < last && alive; ++j) {
                    const long long mine = row;
                    row = look_up(j + 1);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (!wait_empty()) { alive = false; break; }
                        const uint32_t dst = ring + (at % S::kSlots) * S::kBlock;
                        const uint8_t *pool = kv ? a.kv.v : a.kv.k;
#pragma unroll
                        for (int i = 0; i < kLoads; ++i) {
                            const int x = i * 32 + lane, key = w * kKeysW + x / kChunks, ch = x % kChunks;
                            const long long r = __shfl_sync(0xffffffffu, mine, x / kChunks);
                            cp_async16_zero_fill(dst + (ch >> 3) * (kN * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4),
                                                 pool + (size_t)(r < 0 ? 0 : r) * (2 * D) + ch * 16, r >= 0);
                        }
                        cp_async_commit();
                        ++at;
                        cp_async_wait<2>();
                        if (at - 2 > told) hand_over(at - 2);
                    }
                }
            }
            u = line.behind();
            if (u >= line.end) break;
            line.next();
        }
        cp_async_wait<0>();
        hand_over(at);
    } else {
        // ================================ mma ====================================================
        uint32_t p_phase = 0, q_phase = 0;                 // a bit per slot, per tile
        int at = 0;                                        // ring blocks so far (keys and values alternate)
        const bool lead = elect_one();
        auto score = [&](int t, int slot, int blk) {       // S = Q K^T
            const uint32_t k_smem = ring + (blk % S::kSlots) * S::kBlock;
            if (lead) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_f16_ss(tmem + kSlotCol + slot * 128,
                               desc_sw128(q_smem + t * S::kQ + (k >> 2) * (kRowsTile * 128) + (k & 3) * 32, 16),
                               desc_sw128(k_smem + (k >> 2) * (kN * 128) + (k & 3) * 32, 16), kQkDesc, k > 0);
                tc_commit(s_full(slot));
            }
        };
        auto weigh = [&](int t, int slot, int blk, bool fresh) {   // O (+)= P V
            const uint32_t v_smem = ring + (blk % S::kSlots) * S::kBlock;
            if (lead) {
#pragma unroll
                for (int z = 0; z < TERMS; ++z) {
                    const uint32_t p = tmem + kSlotCol + slot * 128 + (z ? 32 + 32 * z : 0);
#pragma unroll
                    for (int k = 0; k < kN / 16; ++k)
                        mma_f16_ts(tmem + t * D, p + k * 8, desc_sw128(v_smem + k * 2048, kN * 128), kPvDesc,
                                   !(fresh && z == 0 && k == 0));
                }
                tc_commit(o_done(t));
            }
        };
        bool alive = true;
        int ready = 0;                                     // ring blocks known to be full
        auto have = [&](int blk) {                         // block number blk has landed
            if (blk < ready) return true;
            if (!wait(full(blk % S::kSlots), (blk / S::kSlots) & 1)) return false;
            ready = blk + 1;
            return true;
        };
        auto free_block = [&](int blk) {
            if (lead) tc_commit(empty(blk % S::kSlots));
        };
        for (long long u = line.begin; alive;) {
            const int first = line.first_unit(u), last = line.last_unit();
            if (last <= first) break;
            int end[kT];
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                end[t] = tile_end(t, last);
                if (alive && first < end[t]) {
                    alive = wait(q_full(t), q_phase >> t & 1);
                    q_phase ^= 1u << t;
                }
            }
            if (!alive) break;
            alive = have(at);
            if (!alive) break;
            tc_fence_after();
#pragma unroll
            for (int t = 0; t < kT; ++t)
                if (first < end[t]) score(t, kT == 2 ? t : 0, at);
            free_block(at);
            for (int j = first; j < last && alive; ++j, at += 2) {
                const int v_blk = at + 1, k_blk = at + 2;
                if constexpr (kT == 1) {
                    const int slot = (j - first) & 1;
                    if (j + 1 < last) {
                        if (!have(k_blk)) { alive = false; break; }
                        tc_fence_after();
                        score(0, slot ^ 1, k_blk);
                        free_block(k_blk);
                    }
                    if (!wait(p_full(slot), p_phase >> slot & 1) || !have(v_blk)) { alive = false; break; }
                    p_phase ^= 1u << slot;
                    tc_fence_after();
                    weigh(0, slot, v_blk, j == first);
                } else {
#pragma unroll
                    for (int t = 0; t < kT; ++t) {
                        if (alive && j < end[t]) {
                            if (!wait(p_full(t), p_phase >> t & 1) || !have(v_blk)) {
                                alive = false;
                            } else {
                                p_phase ^= 1u << t;
                                tc_fence_after();
                                weigh(t, t, v_blk, j == first);
                            }
                        }
                        if (alive && j + 1 < end[t]) {
                            if (!have(k_blk)) {
                                alive = false;
                            } else {
                                tc_fence_after();
                                score(t, t, k_blk);
                            }
                        }
                    }
                    if (!alive) break;
                    if (j + 1 < last) free_block(k_blk);
                }
                free_block(v_blk);
            }
            u = line.behind();
            if (u >= line.end) break;
            line.next();
        }
        // no product runs on and no arrival is under way when the CTA ends, whether or not a wait gave up
        if (lead) tc_commit(drained);
        mbar_wait_bounded(drained, 0, a.kv.status, 24, a.limit_ns);
        __syncwarp();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Joins the tiles that were cut between CTAs: blockIdx.x = the CTA that a tile starts in, blockIdx.y =
// 16 of its dims, a thread per row.
template <int D, int TILES, bool OUT_BF16>
__global__ void __launch_bounds__(TILES * 128) attn_join_kernel(const AttnArgs a, const JoinTile *joins) {
    pdl_wait();
    pdl_trigger();
    const JoinTile jt = joins[blockIdx.x];
    if (!jt.count) return;
    const int t = threadIdx.x >> 7, row = threadIdx.x & 127, d0 = blockIdx.y * 16;
    const long long rho = (long long)jt.m * (TILES * 128) + threadIdx.x;
    if (rho >= (long long)jt.n * a.group) return;
    auto part = [&](int c) {
        const int slot = c == jt.c0 ? jt.slot0 : 2 * c;
        return a.part + (size_t)(slot * TILES + t) * (D + 2) * kRowsTile + row;
    };
    float m = -INFINITY;
    for (int c = jt.c0; c <= jt.c1; ++c) m = fmaxf(m, __ldcg(part(c) + D * kRowsTile));
    float l = 0.0f, o[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = 0.0f;
    for (int c = jt.c0; c <= jt.c1; ++c) {
        const float *p = part(c);
        const float mc = __ldcg(p + D * kRowsTile);
        if (mc == -INFINITY) continue;                 // no key of this part is seen by the row
        const float f = exp2_approx(mc - m);
        l = fmaf(__ldcg(p + (D + 1) * kRowsTile), f, l);
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] = fmaf(__ldcg(p + (size_t)(d0 + x) * kRowsTile), f, o[x]);
    }
    const float f = l > 0.0f ? __fdiv_rn(a.kv.v_scale, l) : (l == l ? 0.0f : l);
    const int tok = (int)(rho / a.group), h = jt.g * a.group + (int)(rho % a.group);
    const size_t to = (size_t)(jt.t0 + tok) * a.ldo + (size_t)h * D + d0;
#pragma unroll
    for (int x = 0; x < 16; x += 4) {
        if constexpr (OUT_BF16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + to + x) =
                make_uint2(pack_bf16(o[x] * f, o[x + 1] * f), pack_bf16(o[x + 2] * f, o[x + 3] * f));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to + x) =
                make_float4(o[x] * f, o[x + 1] * f, o[x + 2] * f, o[x + 3] * f);
    }
}

template <int D, bool E4M3, int TERMS>
void launch(const AttnArgs &a, int sms) {
    using S = TileShape<D, E4M3, TERMS>;
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(attn_tile_kernel<D, E4M3, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        set = true;
    }
    JoinTile *joins = reinterpret_cast<JoinTile *>(a.part + (size_t)2 * sms * S::kTiles * (D + 2) * kRowsTile);
    launch_pdl(attn_tile_kernel<D, E4M3, TERMS>, dim3(sms), dim3(S::kThreads), (size_t)S::kSmem, a, joins);
    TQ_LAUNCH_CHECK("attn_tile_kernel");
    launch_pdl(attn_join_kernel<D, S::kTiles, TERMS == 1>, dim3(sms, D / 16), dim3(S::kTiles * 128), 0, a, (const JoinTile *)joins);
    TQ_LAUNCH_CHECK("attn_join_kernel");
}
template <int D>
void launch_dim(const AttnArgs &a, bool e4m3, int sms) {
    if (a.out_bf16) e4m3 ? launch<D, true, 1>(a, sms) : launch<D, false, 1>(a, sms);
    else e4m3 ? launch<D, true, 2>(a, sms) : launch<D, false, 3>(a, sms);
}

}  // namespace

size_t attn_tile_part_floats(int sms) {
    // two parts per CTA of 256 rows x (128 + 2), or 128 x (256 + 2), and the join kernel's list
    return (size_t)2 * sms * 2 * (128 + 2) * kRowsTile + (size_t)sms * sizeof(JoinTile) / sizeof(float);
}

void launch_attn_tile(const AttnArgs &a, bool e4m3, int sms) {
    if (a.kv.dim == 64) launch_dim<64>(a, e4m3, sms);
    else if (a.kv.dim == 128) launch_dim<128>(a, e4m3, sms);
    else launch_dim<256>(a, e4m3, sms);
}

}  // namespace tq
