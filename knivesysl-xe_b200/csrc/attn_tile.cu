// attn_tile.cu — attention of chunks of new tokens over a paged cache on tcgen05 (x_attn_paged).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m)
//
// A tile is 128 packed query rows (new token x query head) of one key/value head. A CTA carries two of
// them for bf16 outputs at dims 64 and 128, so that the tensor core multiplies for one while the other's
// probabilities are computed, else one: dim 256 and the lower terms of fp32 outputs need the tensor
// memory. Each tile has its own scores S and sums O there. Roles:
//   softmax  one warpgroup per tile, a thread per row: its queries into shared memory (the next tile's
//            under the end of the last), then per block of 64 keys S -> running maximum -> P, written over
//            S as the next product's A operand. Where a CTA has one tile, two warpgroups take turns at its
//            blocks; the maximum passes from one to the other through shared memory, the sums are added
//            at the end
//   load     the blocks of keys and values, page by page, into a ring in shared memory: one warp that
//            issues TMA copies of 8 to 64 rows, or, where pages are no multiple of 8 or the cache is
//            e4m3 (which becomes fp16 on the way), four warps through their registers
//   mma      a warp per tile: S = Q K^T and O += P V, and the barriers that free the ring. Issuing the
//            products of two tiles takes one thread longer (2060 clocks per 64 keys at dim 128) than the
//            tensor core needs for them (1310)
// O is rescaled only when a row's maximum grows by more than 2^8: until then probabilities are up to
// 2^8 instead of 1, which costs no precision, and the rescaling pass over O hardly ever runs. fp16
// probabilities (e4m3 cache) are 2^11 times as large, for fp16's range, and there it is 2^4 (2^14 and 2^1: the
// chunks that kSeg's comment times take 246 us over an e4m3 cache of dim 128, instead of 218).
//
// What bounds it. bf16 outputs: the products of two tiles and 64 keys take 1024 clocks at dim 128, their
// 16384 exponentials as long on the special-function units, next to maxima, sums and packing on the same
// four warps a tile: the softmax warpgroups set the pace. One pair of exponentials in four goes to the FMA
// pipe. 4096 new tokens on as many (40 query, 8 key/value heads of 128): 470 us in a run of that call alone = 0.66 of the
// measured bf16 rate by operations (311 us). fp32 outputs carry P in three terms, four products instead of two: a
// batch of chunks and decodes takes 278 us, 0.40 of the rate by the operations issued (110 us); there the split of P
// into terms, 12 instructions a pair, takes longer than the products, and there is one row tile a CTA. With one
// warpgroup a tile it took 30 us more.
//
// Work is cut into equal stretches of key blocks, one per SM (Line, kv.cuh): a causal batch of any
// lengths loads all SMs alike. A tile cut between CTAs leaves (m, sum, O) of each part in global
// memory, and a second, small kernel joins them in the order of the keys.
//
// Roundings: as in attn_stream.cu. Every 256 to 8192 keys (kSeg) the sums O are added to fp32 sums outside tensor memory.
#include "attn.cuh"
#include "tc.cuh"


#include <algorithm>
#include <type_traits>

namespace tq {

namespace {

constexpr int kRowsTile = 128;
// How the load warps bring a block in.
enum Load { kTma, kRegs, kRegsE4m3 };
constexpr int kCubic = 1;             // of four pairs of exponentials, those that the FMA pipe computes (0, 1, 2, 3: 480, 462, 481, 522 us at 4096 tokens, before the sums left tensor memory)

template <int D, Load LOAD, int TERMS>
struct TileShape {
    static constexpr int kLoadWarps = LOAD == kTma ? 1 : 4;
    // Three terms of P: the second and third add to sums of their own, where tensor memory has room for them beside one
    // row tile. The tensor core cuts an fp32 sum off instead of rounding it, 12 times per 64 keys in one sum for all
    // terms, 4 times in the first term's own (4000 keys: off by 2e-6 of a row with one sum).
    static constexpr bool kLow = TERMS == 3 && D <= 128;
    static constexpr int kTiles = D <= 128 && !kLow ? 2 : 1;        // row tiles of a CTA
    static constexpr int kRows = kRowsTile * kTiles;
    static constexpr int kKeys = 64;                                // of a block
    // Score buffers of a tile. With two, the scores of block j + 1 lie ready when the probabilities of
    // block j are done; more terms of P leave room for one only.
    static constexpr int kBuf = kTiles == 1 || TERMS == 1 ? 2 : 1;
    static constexpr int kSlotCols = 256 / (kTiles * kBuf);
    // Blocks that O sums up in tensor memory before it goes to fp32 sums outside. The tensor core cuts an fp32 sum off, by up
    // to 2^-23 of it, twice in a step of 16 keys: n cuts of a sum that grows evenly take n 2^-24. fp32 outputs: 128 cuts at
    // most, and 4e-6 was the most measured; without it 35000 keys in a row lose 1.5e-4 (two terms), 1.8e-4 (lower terms
    // apart) or 4e-4 (three terms in one sum). bf16 outputs: 140000 keys lost 8e-4 of themselves. Chunks of 1024 and 512
    // tokens on 3000 and 1500, fp32: 189 -> 203 us at dim 128, 126 -> 134 at 64, 197 -> 249 at 256, where a sum of all
    // three terms has to leave every 256 keys.
    static constexpr int kSeg = TERMS == 1 ? 128 : (kLow ? 16 : (TERMS == 2 ? 8 : 4));
    static constexpr int kBlock = kKeys * D * 2;                    // bytes of keys, or of values
    static constexpr int kRing = 131072 / kBlock > 8 ? 8 : 131072 / kBlock;
    static constexpr int kQ = kRowsTile * D * 2;                    // bytes of a tile's queries
    static constexpr int kSmem = kTiles * kQ + kRing * kBlock + 1024;
    static constexpr int kSoftmax = 256;                            // threads: a warpgroup per tile, or two that share one
    static constexpr int kThreads = kSoftmax + kLoadWarps * 32 + kTiles * 32;
};

// 128-byte swizzle: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7), groups of 8 rows 1024
// bytes apart (SBO). K-major operands step 32 bytes per k16; MN-major ones (values: the summed
// dimension runs over rows) have their next 64 columns LBO bytes further on.
// desc_lo: the low word, start address and LBO; the rest is the same for all (SBO, version 1, swizzle).
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFFu) >> 4) | (lbo >> 4) << 16; }
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
    return (uint64_t)lo | (uint64_t)((1024u >> 4) | 1u << 14 | 2u << 29) << 32;
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
// A box of rows of 128 bytes to shared memory, 128-byte swizzled; rows outside the tensor come as zeros.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A row tile's sums in global memory, four dims of a row together: neighbouring threads (rows) take neighbouring 16 bytes.
// Behind them, as if they were four more, the row's maximum and its sum of weights.
template <int D>
constexpr int kPartFloats = (D + 4) * kRowsTile;
__device__ __forceinline__ float *part_at(float *row, int dim) { return row + dim * kRowsTile; }      // row: the first of its places
// Written, added to and read by one thread, past L1.
__device__ __forceinline__ void st_sums(float *p, float4 v) {
    asm volatile("st.relaxed.gpu.global.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void add_sums(float *p, float4 v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ float4 ld_sums(const float *p) {
    float4 v;
    asm volatile("ld.relaxed.gpu.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

// COLS dims of a row's sums leave tensor memory for those in global memory (the tile's place among the parts, whether or
// not it is cut): stored the first time (`once`), then added. Adding without reading has nothing to wait for; one thread's
// additions to an address keep their order. The sums outside go by the maximum *ref, those in tensor memory by `top`, which
// is no smaller; grown by more than 2^8, it scales the former first.
template <int COLS>
__device__ __forceinline__ void flush_sums(float *part, uint32_t o_col, float *ref_at, bool once, float top) {
    float ref = once ? top : *ref_at;
    if (__any_sync(0xffffffffu, top > ref + 8.0f)) {
        const float by = top == -INFINITY ? 1.0f : exp2_approx(ref - top);
#pragma unroll 2
        for (int x = 0; x < COLS; x += 4) {
            float4 v = ld_sums(part_at(part, x));
            v.x *= by; v.y *= by; v.z *= by; v.w *= by;
            st_sums(part_at(part, x), v);
        }
        ref = top;
    }
    *ref_at = ref;
    const float f = top == -INFINITY ? 0.0f : exp2_approx(top - ref);
#pragma unroll 1
    for (int x = 0; x < COLS; x += 32) {
        uint32_t v[32];
        tmem_ld32(o_col + x, v);
        tmem_wait32(v);
#pragma unroll
        for (int y = 0; y < 32; y += 4) {
            const float4 z = make_float4(__uint_as_float(v[y]) * f, __uint_as_float(v[y + 1]) * f, __uint_as_float(v[y + 2]) * f,
                                         __uint_as_float(v[y + 3]) * f);
            if (once) st_sums(part_at(part, x + y), z);
            else add_sums(part_at(part, x + y), z);
        }
    }
}

// The same out of line, where the block loop has no registers to spare: a call costs the loop some as well. Measured, inline
// and called: 2048 new tokens, dim 128, bf16 in and out 87 and 98 us; the chunks of kSeg's times at dim 256, fp32 249 and 258,
// bf16 162 and 156, dim 128 over e4m3, bf16, 166 and 156; else within 1 %.
template <int COLS>
static __device__ __noinline__ void flush_sums_call(float *part, uint32_t o_col, float *ref_at, bool once, float top) {
    flush_sums<COLS>(part, o_col, ref_at, once, top);
}

__device__ __forceinline__ float max3(float x, float y, float z) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
    return d;
}
// 2^x for a pair, x <= 15, by the FMA pipe: x = n + f with |f| <= 1/2 (n rounded off by adding 1.5 x 2^23),
// 2^f a cubic with the smallest relative error on that interval, 7.5e-5 (fitted by Remez exchange),
// times 2^n (a product, not an addition to the exponent: a NaN stays one). x below -126 (-inf too: a masked key) gives 2^-126
// or so, which is nothing beside the row's largest, 1.
__device__ __forceinline__ void exp2_cubic(f32x2 x, float &e0, float &e1) {
    float x0, x1, r0, r1;
    unpack2(x, x0, x1);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-126.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-126.0f));
    x = pack2(x0, x1);
    const f32x2 r = add2(x, pack2(kMagicF, kMagicF));
    const f32x2 f = fma2(add2(r, pack2(-kMagicF, -kMagicF)), pack2(-1.0f, -1.0f), x);
    f32x2 p = fma2(pack2(0.0551716691f, 0.0551716691f), f, pack2(0.242611122f, 0.242611122f));
    p = fma2(p, f, pack2(0.693260985f, 0.693260985f));
    p = fma2(p, f, pack2(0.999928074f, 0.999928074f));
    unpack2(r, r0, r1);
    unpack2(mul2(p, pack2(__uint_as_float((__float_as_uint(r0) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(r1) << 23) + 0x3f800000u))), e0, e1);
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

template <int D, Load LOAD, int TERMS>
__global__ void __launch_bounds__((TileShape<D, LOAD, TERMS>::kThreads), 1)
    attn_tile_kernel(const AttnArgs a, JoinTile *joins, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
    using S = TileShape<D, LOAD, TERMS>;
    constexpr bool E4M3 = LOAD == kRegsE4m3;
    constexpr int kT = S::kTiles, kN = S::kKeys;
    constexpr bool OUT_BF16 = TERMS == 1;
    constexpr float kLift = E4M3 ? 11.0f : 0.0f, kLag = E4M3 ? 4.0f : 8.0f;    // of the probabilities' exponents, of the maximum's
    constexpr int kBuf = S::kBuf, kScores = kT * kBuf;
    constexpr uint32_t kSlotCol = 256;                 // tensor memory: O tiles (and the lower terms' sums), then the slots of S and P
    constexpr uint32_t kQkDesc = idesc_f16(128, kN, !E4M3, false), kPvDesc = idesc_f16(128, D, !E4M3, true);

    extern __shared__ uint8_t smem_raw[];
    __shared__ long long s_scan[S::kThreads / 32 + 3];
    __shared__ __align__(8) uint64_t s_bar[2 * S::kRing + 2 * kScores + 3 * kT + 4];
    __shared__ uint32_t s_tmem;
    __shared__ float s_c[128], s_m[128], s_ml[2][2][128];        // one tile: factor, maximum of each row; (m, l) of each warpgroup
    __shared__ float s_ref[S::kSoftmax];               // of a thread's row: the maximum that its sums outside tensor memory go by
    __shared__ int s_gave_up, s_stop;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    const int G = a.group;
    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_smem = base, ring = base + kT * S::kQ;
    const uint32_t bars = smem_u32(s_bar);
    auto full = [&](int i) { return bars + 8 * i; };                        // ring slot holds a block
    auto empty = [&](int i) { return bars + 8 * (S::kRing + i); };         // and may be written again
    auto s_full = [&](int i) { return bars + 8 * (2 * S::kRing + i); };    // slot i holds scores
    auto p_full = [&](int i) { return bars + 8 * (2 * S::kRing + kScores + i); };
    auto q_full = [&](int i) { return bars + 8 * (2 * S::kRing + 2 * kScores + i); };
    auto o_done = [&](int i) { return bars + 8 * (2 * S::kRing + 2 * kScores + kT + i); };   // a P V product of tile i is complete
    auto o_last = [&](int i) { return bars + 8 * (2 * S::kRing + 2 * kScores + 2 * kT + i); };   // the last one of a stretch's tile
    const uint32_t drained = bars + 8 * (2 * S::kRing + 2 * kScores + 3 * kT);       // all products and their arrivals are done

    const uint32_t m_ready = drained + 16;             // one tile: the maximum up to a block is in s_m
    const uint32_t flushed = drained + 24;             // one tile: the second warpgroup's share of O has left tensor memory
    const uint32_t landed = drained + 8;               // a block that the load warp has to complete itself

    if (tid == 0) {
        mbar_init(drained, kT);
        mbar_init(landed, 1);
        mbar_init(m_ready, 4);
        mbar_init(flushed, 4);
        for (int i = 0; i < S::kRing; ++i) {
            mbar_init(full(i), S::kLoadWarps);
            mbar_init(empty(i), kT);
        }
        for (int i = 0; i < kScores; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), 4);
        }
        for (int i = 0; i < kT; ++i) {
            mbar_init(q_full(i), S::kSoftmax / 32 / kT);
            mbar_init(o_done(i), 1);
            mbar_init(o_last(i), 1);
        }
        mbar_init_fence();
        s_gave_up = 0;
    }
    pdl_wait();
    pdl_trigger();
    Line<S::kRows> line(a.kv, G, kN, 4);
    const bool work = line.template locate<S::kThreads>(s_scan, cta, gridDim.x);
    if (tid == 0) joins[cta].count = 0;
    if (!work) return;
    constexpr int kMmaWarp = S::kSoftmax / 32 + S::kLoadWarps;
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
        constexpr int kGroups = 2 / kT;                    // warpgroups of a tile
        const int t = kT == 2 ? warp >> 2 : 0, wg = kT == 2 ? 0 : warp >> 2, row = tid & 127;
        const uint32_t lane_col = tmem + ((uint32_t)(warp & 3) << 21);
        const uint32_t o_col = lane_col + t * D;
        uint32_t s_phase = 0, blocks_done = 0, tiles_done = 0;     // a bit per slot; blocks and tiles of this tile so far
        bool alive = true;                                 // no wait of this warp gave up
        // A stretch's tile as this thread sees it.
        struct Part {
            int first, last, end;                          // units, and the end of this row tile's own
            int limit, low;                                // last key that the row sees, that every row sees
            bool live, whole;
            long long query;                               // the row's place in q, -1 for none
            size_t to;                                     // and in the output
            float *part;                                   // where the tile is cut: its place in the parts
            long long behind;
        };
        auto describe = [&](long long u) {
            Part x;
            const KvRequest &req = line.q;
            x.first = line.first_unit(u);
            x.last = line.last_unit();
            x.end = tile_end(t, x.last);
            const int rho = line.m * S::kRows + t * kRowsTile + row, tok = rho / G;
            x.live = row < tile_rows(t);
            x.limit = x.live ? req.total - req.n + tok : -1;
            x.low = req.total - req.n + (line.m * S::kRows + t * kRowsTile) / G;
            x.whole = x.first == 0 && x.last == line.units;
            x.query = x.live ? ((long long)(req.t0 + tok) * a.q_heads + line.g * G + rho % G) * D : -1;
            x.to = (size_t)(req.t0 + tok) * a.ldo + (size_t)(line.g * G + rho % G) * D;
            const int slot = 2 * cta + (u == line.begin ? 0 : 1);
            x.part = a.part + (size_t)(slot * kT + t) * kPartFloats<D> + row * 4;
            x.behind = line.behind();
            if (tid == 0 && x.first == 0 && x.last > 0 && !x.whole)      // the tile starts here and goes on: its parts
                joins[cta] = JoinTile{req.t0, req.n, line.g, line.m, cta, line.cta_of(x.behind - 1), slot, 1};
            return x;
        };
        // The queries of a tile into shared memory, once the products with the last ones are complete; the factor
        // of the row's scores.
        auto load_q = [&](const Part &x) {
            float c = fabsf(a.c);
            // ---- the warp's 32 rows of queries, turned by the sign of the scale, whole rows per load
            const uint32_t flip = a.c < 0.0f ? 0x80008000u : 0u, keep = a.c != 0.0f ? 0xffffffffu : 0u;
            const uint32_t q_tile = q_smem + t * S::kQ;
            constexpr int kQChunks = D / 8;            // 16-byte chunks of a row
            constexpr int kShare = kQChunks / kGroups, kAtOnce = kShare < 8 ? kShare : 8;
            uint4 v[kAtOnce];
#pragma unroll
            for (int x0 = wg * kShare; x0 < (wg + 1) * kShare; x0 += kAtOnce) {
#pragma unroll
                for (int n = 0; n < kAtOnce; ++n) {
                    const int i = (x0 + n) * 32 + lane;
                    const long long from = __shfl_sync(0xffffffffu, x.query, i / kQChunks);
                    v[n] = from >= 0 ? __ldg(reinterpret_cast<const uint4 *>(a.q + from) + i % kQChunks) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int n = 0; n < kAtOnce; ++n) {
                    const int i = (x0 + n) * 32 + lane, r = (warp & 3) * 32 + i / kQChunks, ch = i % kQChunks;
                    st_shared16(q_tile + (ch >> 3) * (kRowsTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                                make_uint4((v[n].x ^ flip) & keep, (v[n].y ^ flip) & keep, (v[n].z ^ flip) & keep,
                                           (v[n].w ^ flip) & keep));
                }
            }
            if constexpr (E4M3) {
                // own row: to fp16, times the power of two that takes its largest value to [2^9, 2^10)
                if constexpr (kGroups == 2) named_bar_sync(2, 256);
                else __syncwarp();
                if (wg == 0) {
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
                    s_c[row] = c;
                }
                if constexpr (kGroups == 2) {
                    named_bar_sync(2, 256);
                    c = s_c[row];
                }
            }
            if (!(c > 0.0f)) c = 1.17549435e-38f;      // scores of no size: any factor above 0
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(t));
            return c;
        };
        Part cur = describe(line.begin);
        if (cur.last <= cur.first) cur.end = 0;            // the stretch ends before the tile's first unit
        float c = cur.first < cur.end ? load_q(cur) : 0.0f;
        while (cur.last > cur.first) {
            const int limit = cur.limit, low = cur.low;
            const bool more = cur.behind < line.end, live = cur.live;
            float m = -INFINITY, l = 0.0f, c_next = 0.0f;
            // This warpgroup's share of O, which has the maximum `top`, leaves for sums outside (see flush_sums).
            auto flush = [&](bool once, float top) {
                float *const part = part_at(cur.part, wg * (D / kGroups));
                const uint32_t col = o_col + wg * (D / kGroups);
                if constexpr (LOAD == kTma && (D <= 128 || TERMS > 1)) flush_sums<D / kGroups>(part, col, s_ref + tid, once, top);
                else flush_sums_call<D / kGroups>(part, col, s_ref + tid, once, top);
            };
            Part next = cur;
            next.last = next.first;                        // none
            auto prepare = [&]() {                         // the stretch's next tile: its queries are on their way under this one's end
                if (!more) return;
                line.next();
                next = describe(cur.behind);
                if (next.last > next.first && next.first < next.end) c_next = load_q(next);
            };
            if (cur.first < cur.end) {
                // Every kSeg blocks O leaves for fp32 sums outside. A warpgroup with a tile of its own does that between two
                // loops over blocks, two that share one from within.
                for (int seg = cur.first; seg < cur.end && alive;) {
                    const int seg_end = kGroups == 1 ? min(cur.end, seg + S::kSeg) : cur.end;
                    for (int j = seg + wg; j < seg_end && alive; j += kGroups) {
                        const int slot = t * kBuf + (kBuf == 2 ? (j - seg) & 1 : 0);
                        const uint32_t s_col = lane_col + kSlotCol + slot * S::kSlotCols;
                        if (!wait(s_full(slot), s_phase >> slot & 1)) { alive = false; break; }
                        s_phase ^= 1u << slot;
                        tc_fence_after();
                        const int key0 = j * kN;
                        const bool anew = kGroups == 2 && j > seg && (j - seg) % S::kSeg == 0;    // this block's product starts O anew
                        const bool cut = key0 + kN - 1 > low;
                        // ---- maximum of the block
                        uint32_t v0[32], v1[32];
                        tmem_ld32(s_col, v0);
                        tmem_ld32(s_col + 32, v1);
                        tmem_wait32(v0);
                        tmem_wait32(v1);
                        if (cut) {
#pragma unroll
                            for (int y = 0; y < 32; ++y) {
                                if (key0 + y > limit) v0[y] = 0xff800000u;
                                if (key0 + 32 + y > limit) v1[y] = 0xff800000u;
                            }
                        }
                        float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                        for (int y = 0; y < 32; y += 2) {
                            mx = max3(mx, __uint_as_float(v0[y]), __uint_as_float(v0[y + 1]));
                            mx1 = max3(mx1, __uint_as_float(v1[y]), __uint_as_float(v1[y + 1]));
                        }
                        mx = fmaxf(mx, mx1);
                        mx *= c;
                        const uint32_t done = blocks_done + (j - seg);       // blocks before this one
                        float before = m;                      // the maximum that O and the blocks before have
                        if constexpr (kGroups == 2) {
                            before = -INFINITY;
                            if (j > seg) {
                                if (!wait(m_ready, (done - 1) & 1)) { alive = false; break; }
                                before = s_m[row];
                            }
                        }
                        const bool grows = mx > before + kLag;
                        const float now = grows ? mx : before;
                        if constexpr (kGroups == 2) {
                            s_m[row] = now;
                            __syncwarp();
                            if (lane == 0) mbar_arrive(m_ready);
                        }
                        if (j > seg && (S::kLow || !anew) && __any_sync(0xffffffffu, grows)) {
                            // The product of block j - 1 must be in O. That of j - 2 is (the scores of block j were
                            // multiplied behind it), so the barrier is at most one phase behind.
                            if (!wait(o_done(t), (done - 1) & 1)) { alive = false; break; }
                            tc_fence_after();
                            const float f = grows ? exp2_approx(before - mx) : 1.0f;
                            // a short loop: unrolled, its registers push others of the block loop out
#pragma unroll 1
                            for (int x = anew ? D : 0; x < (S::kLow ? 2 * D : D); x += 16) {
                                uint32_t v[16];
                                tmem_ld16(o_col + x, v);
                                tmem_wait_ld16(v);
#pragma unroll
                                for (int y = 0; y < 16; ++y) v[y] = __float_as_uint(__uint_as_float(v[y]) * f);
                                tmem_st16(o_col + x, v);
                            }
                        }
                        // this thread's sum so far has the maximum that it last saw
                        if (now != m) {
                            l *= exp2_approx(m - now);
                            m = now;
                        }
                        const float off = m == -INFINITY ? 0.0f : kLift - m;
                        // ---- probabilities, over the scores
                        f32x2 sum = pack2(0.0f, 0.0f);
                        const f32x2 c2 = pack2(c, c), off2 = pack2(off, off);
                        auto weights = [&](const uint32_t (&sc)[32], int x) {
                            uint32_t w[TERMS][16];
#pragma unroll
                            for (int y = 0; y < 32; y += 2) {
                                float p0, p1;
                                const f32x2 z = fma2(pack2(__uint_as_float(sc[y]), __uint_as_float(sc[y + 1])), c2, off2);
                                if (TERMS == 1 && (y & 7) >= 8 - 2 * kCubic) {
                                    exp2_cubic(z, p0, p1);
                                } else {
                                    unpack2(z, p0, p1);
                                    p0 = exp2_approx(p0);
                                    p1 = exp2_approx(p1);
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
                        };
                        weights(v0, 0);
                        weights(v1, 32);
                        if (anew) {
                            // O holds the blocks up to j - 1 (the barrier is at most one phase behind, as above)
                            if (!wait(o_done(t), (done - 1) & 1)) { tmem_wait_st(); alive = false; break; }
                            tc_fence_after();
                            flush(j - seg == S::kSeg, before);
                        }
                        float l0, l1;
                        unpack2(sum, l0, l1);
                        l += l0 + l1;
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_full(slot));
                        if constexpr (kGroups == 2) {
                            // The other warpgroup's block starts O anew. Blocks take turns and kSeg is even, so this is always the
                            // second one. O holds the blocks up to this one; the barrier may be two phases behind.
                            if (j + 1 < seg_end && (j + 1 - seg) % S::kSeg == 0) {
                                if (!wait(o_done(t), (done - 1) & 1) || !wait(o_done(t), done & 1)) { alive = false; break; }
                                tc_fence_after();
                                flush(j + 1 - seg == S::kSeg, now);
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(flushed);
                            }
                        }
                    }
                    blocks_done += seg_end - seg;
                    if (kGroups == 1 && seg_end < cur.end && alive) {
                        // the product of the last block may be two phases away
                        if (!wait(o_done(t), blocks_done & 1) || !wait(o_done(t), (blocks_done - 1) & 1)) { alive = false; break; }
                        tc_fence_after();
                        flush(seg == cur.first, m);
                    }
                    seg = seg_end;
                }
                // With a tile of its own, a warpgroup has seen the scores of the last block: no product reads the
                // queries any more. Of two, one may not have: there the last product is waited for first.
                if constexpr (kGroups == 1) prepare();
                alive = alive && wait(o_last(t), tiles_done++ & 1);
                tc_fence_after();
                if constexpr (kGroups == 2) {
                    s_ml[wg][0][row] = m;
                    s_ml[wg][1][row] = l;
                    named_bar_sync(2, 256);
                    const float mo = s_ml[wg ^ 1][0][row], lo = s_ml[wg ^ 1][1][row], both = fmaxf(m, mo);
                    if (both != -INFINITY) l = (m == -INFINITY ? 0.0f : l * exp2_approx(m - both)) + (mo == -INFINITY ? 0.0f : lo * exp2_approx(mo - both));
                    m = both;
                    prepare();
                }
            } else {
                prepare();
            }
            // ---- the tile's rows, or this CTA's part of them (whatever they hold, if a wait gave up)
            const bool outside = cur.end - cur.first > S::kSeg;
            const float f_ref = outside && s_ref[tid] != -INFINITY ? exp2_approx(s_ref[tid] - m) : 0.0f;
            auto load_o = [&](int x, uint32_t (&v)[32]) {
                tmem_ld32(o_col + x, v);
                tmem_wait32(v);
                if constexpr (S::kLow) {
                    uint32_t w[32];
                    tmem_ld32(o_col + D + x, w);
                    tmem_wait32(w);
#pragma unroll
                    for (int y = 0; y < 32; ++y) v[y] = __float_as_uint(__uint_as_float(v[y]) + __uint_as_float(w[y]));
                }
                if (outside) {
#pragma unroll
                    for (int y = 0; y < 32; y += 4) {
                        const float4 z = ld_sums(part_at(cur.part, x + y));
                        v[y] = __float_as_uint(fmaf(z.x, f_ref, __uint_as_float(v[y])));
                        v[y + 1] = __float_as_uint(fmaf(z.y, f_ref, __uint_as_float(v[y + 1])));
                        v[y + 2] = __float_as_uint(fmaf(z.z, f_ref, __uint_as_float(v[y + 2])));
                        v[y + 3] = __float_as_uint(fmaf(z.w, f_ref, __uint_as_float(v[y + 3])));
                    }
                }
            };
            if (cur.whole) {
                const float f = l > 0.0f ? __fdiv_rn(a.kv.v_scale, l) : (l == l ? 0.0f : l);
                const size_t to = cur.to;
                if (cur.first < cur.end)
#pragma unroll
                    for (int xx = 0; xx < D / kGroups; xx += 32) {
                        const int x = wg * (D / kGroups) + xx;
                        uint32_t v[32];
                        load_o(x, v);
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
                float *const part = cur.part;
                if (cur.first < cur.end)
#pragma unroll 1
                    for (int xx = 0; xx < D / kGroups; xx += 32) {
                        const int x = wg * (D / kGroups) + xx;
                        uint32_t v[32];
                        load_o(x, v);
#pragma unroll
                        for (int y = 0; y < 32; y += 4)
                            *reinterpret_cast<uint4 *>(part_at(part, x + y)) = make_uint4(v[y], v[y + 1], v[y + 2], v[y + 3]);
                    }
                if (wg == 0) {
                    *reinterpret_cast<float2 *>(part_at(part, D)) = make_float2(m, l);
                }
            }
            tc_fence_before();
            if constexpr (kGroups == 2) {
                // O has been read by both, and both go on or end together: neither leaves the other at a barrier
                if (tid == 0) s_stop = s_gave_up;
                named_bar_sync(2, 256);
                if (s_stop) break;
            } else if (!alive) {
                break;
            }
            cur = next;
            c = c_next;
        }
    } else if (warp < kMmaWarp) {
        // ================================ load ===================================================
        int at = 0;                                        // blocks so far; slot at % kRing
        bool alive = true;
        auto wait_empty = [&]() {
            return at < S::kRing || wait(empty(at % S::kRing), ((at / S::kRing) - 1) & 1);
        };
        if constexpr (LOAD == kTma) {
            uint32_t landings = 0;
            for (long long u = line.begin; alive;) {
                const int first = line.first_unit(u), last = line.last_unit();
                if (last <= first) break;
                const int box = a.box, boxes = kN / box;
                // a lane per box: its first row in the pools; behind the last page's rows (read as zeros) for a bad page
                auto look_up = [&](int j) {
                    const int key = j * kN + lane * box;
                    if (j >= last || lane >= boxes || key >= line.keys) return a.rows;
                    const long long row = kv_row(a.kv, line.r, line.g, key);
                    return row < 0 ? a.rows : (int)row;
                };
                int next = look_up(first);
                for (int j = first; j < last && alive; ++j) {
                    const int row = next;
                    next = look_up(j + 1);
                    const int rest = line.keys - j * kN;       // rows behind the request's last key: whatever the page holds
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (!wait_empty()) { alive = false; break; }
                        const uint32_t dst = ring + (at % S::kRing) * S::kBlock;
                        const bool tail = kv && rest < kN;     // a probability of 0 times that must be 0: zeros instead
                        const uint32_t bar = tail ? landed : full(at % S::kRing);
                        if (lane == 0) mbar_expect_tx(bar, S::kBlock);
                        __syncwarp();
                        if (lane < boxes)
#pragma unroll
                            for (int x = 0; x < D / 64; ++x)
                                tma_load(dst + x * (kN * 128) + lane * box * 128, kv ? &v_map : &k_map, x * 64, row, bar);
                        if (tail) {
                            if (!wait(landed, landings++ & 1)) { alive = false; break; }
                            for (int i = lane; i < (kN - rest) * (D / 8); i += 32)
                                st_shared16(dst + (i & 7) * 16 + (i >> 3) % (D / 64) * (kN * 128) + (rest + (i >> 3) / (D / 64)) * 128,
                                            make_uint4(0, 0, 0, 0));
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(full(at % S::kRing));
                        }
                        ++at;
                    }
                }
                u = line.behind();
                if (u >= line.end) break;
                line.next();
            }
            // the copies in flight end before the CTA does: the products wait for them, unless a wait gave up
            if (!alive)
                for (int i = max(0, at - S::kRing); i < at; ++i)
                    mbar_wait_bounded(full(i % S::kRing), (i / S::kRing) & 1, a.kv.status, 24, a.limit_ns);
            __syncwarp();
        } else {
            constexpr int kKeysW = kN / S::kLoadWarps;         // keys of a warp
            constexpr int kChunks = (E4M3 ? D : 2 * D) / 16;   // of a cached row
            constexpr int kAll = kKeysW * kChunks / 32, kLoads = kAll > 8 ? 8 : kAll;      // loads of a block, in one go
            const int w = warp - S::kSoftmax / 32;
            for (long long u = line.begin; alive;) {
                const int first = line.first_unit(u), last = line.last_unit();
                if (last <= first) break;
                auto look_up = [&](int j) {
                    const int key = j * kN + w * kKeysW + (lane % kKeysW);
                    return j < last && key < line.keys ? kv_row(a.kv, line.r, line.g, key) : -1ll;
                };
                long long row = look_up(first);
                uint4 held[kLoads];
                auto load = [&](const uint8_t *pool, int part) {
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int x = (part * kLoads + i) * 32 + lane;
                        const long long r = __shfl_sync(0xffffffffu, row, x / kChunks);
                        held[i] = r >= 0 ? __ldg(reinterpret_cast<const uint4 *>(pool + ((size_t)r * kChunks + x % kChunks) * 16))
                                         : make_uint4(0, 0, 0, 0);
                    }
                };
                auto store = [&](int part) {
                    const uint32_t dst = ring + (at % S::kRing) * S::kBlock;
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int x = (part * kLoads + i) * 32 + lane, key = w * kKeysW + x / kChunks;
                        if constexpr (E4M3) {              // 16 values -> two chunks of 8 fp16 values
                            const int ch = x % kChunks * 2;
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
                        } else {
                            const int ch = x % kChunks;
                            st_shared16(dst + (ch >> 3) * (kN * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4), held[i]);
                        }
                    }
                };
                // the next block's first loads are under way while this one waits for its slot
                load(a.kv.k, 0);
                for (int j = first; j < last && alive; ++j) {
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (!wait_empty()) { alive = false; break; }
                        store(0);
#pragma unroll
                        for (int part = 1; part < kAll / kLoads; ++part) {
                            load(kv ? a.kv.v : a.kv.k, part);
                            store(part);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(full(at % S::kRing));
                        ++at;
                        if (kv) row = look_up(j + 1);
                        load(kv ? a.kv.k : a.kv.v, 0);
                    }
                }
                u = line.behind();
                if (u >= line.end) break;
                line.next();
            }
        }
    } else {
        // ================================ mma ====================================================
        // One thread does it all: what it spends between two products may be time that the tensor core waits.
        const int t = warp - kMmaWarp;
        if (elect_one()) {
            auto hold = [&](uint32_t bar, uint32_t parity) {
                if (mbar_try_wait(bar, parity)) return true;
                if (*wait.gave_up) return false;
                if (mbar_wait_slow(bar, parity, a.kv.status, 24, a.limit_ns)) return true;
                *wait.gave_up = 1;
                return false;
            };
            uint32_t p_phase = 0, q_phase = 0, flushes = 0;    // a bit per score buffer; queries, flushes so far
            int at = 0;                                    // ring blocks so far (keys and values alternate)
            // descriptors: the word with the address, counted in 16 bytes; a block of the ring, or a tile's
            // queries, is a whole number of those further on
            const uint32_t q_lo = desc_lo(q_smem + t * S::kQ, 16), k_lo = desc_lo(ring, 16), v_lo = desc_lo(ring, kN * 128);
            auto score = [&](int slot, int blk) {          // S = Q K^T
                const uint32_t kd = k_lo + (blk & (S::kRing - 1)) * (S::kBlock >> 4);
                const uint32_t d = tmem + kSlotCol + slot * S::kSlotCols;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_f16_ss(d, desc_of(q_lo + (((k >> 2) * (kRowsTile * 128) + (k & 3) * 32) >> 4)),
                               desc_of(kd + (((k >> 2) * (kN * 128) + (k & 3) * 32) >> 4)), kQkDesc, k > 0);
                tc_commit(s_full(slot));
            };
            auto weigh = [&](int slot, int blk, bool fresh, bool fresh_low, bool closes) {   // O (+)= P V
                const uint32_t vd = v_lo + (blk & (S::kRing - 1)) * (S::kBlock >> 4);
                const uint32_t d = tmem + t * D, p = tmem + kSlotCol + slot * S::kSlotCols;
                // in one sum the lower terms come first: onto a fresh sum they add without loss
#pragma unroll
                for (int zz = 0; zz < TERMS; ++zz) {
                    const int z = S::kLow ? zz : TERMS - 1 - zz;
#pragma unroll
                    for (int k = 0; k < kN / 16; ++k)
                        mma_f16_ts(S::kLow && z ? d + D : d, p + (z ? 32 + 32 * z : 0) + k * 8, desc_of(vd + (k * 2048 >> 4)), kPvDesc,
                                   k || zz > (S::kLow ? 1 : 0) ? 1u : ((S::kLow && z ? fresh_low : fresh) ? 0u : 1u));
                }
                tc_commit(o_done(t));
                if (closes) tc_commit(o_last(t));
            };
            // Every block is waited for and given back, also those that only the other tile's rows see
            auto have = [&](int blk) { return hold(full(blk & (S::kRing - 1)), (blk / S::kRing) & 1); };
            auto free_block = [&](int blk) { tc_commit(empty(blk & (S::kRing - 1))); };
            bool alive = true;
            for (long long u = line.begin; alive;) {
                const int first = line.first_unit(u), last = line.last_unit(), end = tile_end(t, last);
                if (last <= first) break;
                if (first < end) {
                    alive = hold(q_full(t), q_phase & 1);
                    ++q_phase;
                }
                // the first kBuf blocks' scores, then block by block: P V, and the scores of the block that
                // takes over its buffer
                for (int j = first; j < min(first + kBuf, last) && alive; ++j) {
                    const int k_blk = at + 2 * (j - first);
                    alive = have(k_blk);
                    tc_fence_after();
                    if (alive && j < end) score(t * kBuf + (j - first), k_blk);
                    free_block(k_blk);
                }
                for (int j = first; j < last && alive; ++j, at += 2) {
                    const int v_blk = at + 1, k_blk = at + 2 * kBuf, buf = (j - first) & (kBuf - 1), slot = t * kBuf + buf;
                    alive = have(v_blk);
                    if (alive && j < end) {
                        alive = hold(p_full(slot), p_phase >> buf & 1);
                        p_phase ^= 1u << buf;
                        if (kT == 1 && alive && j > first && (j - first) % S::kSeg == 0) alive = hold(flushed, flushes++ & 1);
                        tc_fence_after();
                        if (alive) weigh(slot, v_blk, (j - first) % S::kSeg == 0, j == first, j + 1 == end);
                    }
                    free_block(v_blk);
                    if (alive && j + kBuf < last) {
                        alive = have(k_blk);
                        tc_fence_after();
                        if (alive && j + kBuf < end) score(slot, k_blk);
                        free_block(k_blk);
                    }
                }
                u = line.behind();
                if (u >= line.end) break;
                line.next();
            }
            // no product runs on and no arrival is under way when the CTA ends, whether or not a wait gave up
            tc_commit(drained);
            mbar_wait_bounded(drained, 0, a.kv.status, 24, a.limit_ns);
        }
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
        return a.part + (size_t)(slot * TILES + t) * kPartFloats<D> + row * 4;
    };
    float m = -INFINITY;
    for (int c = jt.c0; c <= jt.c1; ++c) m = fmaxf(m, __ldcg(part_at(part(c), D)));
    float l = 0.0f, o[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = 0.0f;
    for (int c = jt.c0; c <= jt.c1; ++c) {
        float *const p = part(c);
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_at(p, D)));
        const float mc = ml.x;
        if (mc == -INFINITY && ml.y == ml.y) continue; // no key of this part is seen by the row (or only such as give NaN)
        const float f = exp2_approx(mc - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(part_at(p, d0 + x)));
            o[x] = fmaf(v.x, f, o[x]);
            o[x + 1] = fmaf(v.y, f, o[x + 1]);
            o[x + 2] = fmaf(v.z, f, o[x + 2]);
            o[x + 3] = fmaf(v.w, f, o[x + 3]);
        }
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

template <int D, Load LOAD, int TERMS>
void launch(const AttnArgs &a, int sms, const CUtensorMap &k_map, const CUtensorMap &v_map) {
    using S = TileShape<D, LOAD, TERMS>;
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(attn_tile_kernel<D, LOAD, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        set = true;
    }
    JoinTile *joins = reinterpret_cast<JoinTile *>(a.part + (size_t)2 * sms * S::kTiles * kPartFloats<D>);
    launch_pdl(attn_tile_kernel<D, LOAD, TERMS>, dim3(sms), dim3(S::kThreads), (size_t)S::kSmem, a, joins, k_map, v_map);
    TQ_LAUNCH_CHECK("attn_tile_kernel");
    launch_pdl(attn_join_kernel<D, S::kTiles, TERMS == 1>, dim3(sms, D / 16), dim3(S::kTiles * 128), 0, a, (const JoinTile *)joins);
    TQ_LAUNCH_CHECK("attn_join_kernel");
}
template <int D>
void launch_dim(AttnArgs a, bool e4m3, int sms) {
    CUtensorMap k_map{}, v_map{};
    if (e4m3) {
        a.out_bf16 ? launch<D, kRegsE4m3, 1>(a, sms, k_map, v_map) : launch<D, kRegsE4m3, 2>(a, sms, k_map, v_map);
        return;
    }
    // boxes of rows inside one page, in whole swizzle patterns of 8 rows; rows are counted in 32 bits
    const long long rows = (long long)a.kv.pages * a.kv.heads * a.kv.page_size;
    a.box = 64;
    while (a.box > 4 && a.kv.page_size % a.box) a.box /= 2;
    a.rows = rows < 0x7fffffffll ? (int)rows : 0;
    if (a.box >= 8 && a.rows && tensor_map_2d(k_map, a.kv.k, D, rows, a.box) && tensor_map_2d(v_map, a.kv.v, D, rows, a.box))
        a.out_bf16 ? launch<D, kTma, 1>(a, sms, k_map, v_map) : launch<D, kTma, 3>(a, sms, k_map, v_map);
    else
        a.out_bf16 ? launch<D, kRegs, 1>(a, sms, k_map, v_map) : launch<D, kRegs, 3>(a, sms, k_map, v_map);
}

}  // namespace

size_t attn_tile_part_floats(int sms) {
    // two parts per CTA of two row tiles at dim 128, or of one at 256, and the join kernel's list
    return (size_t)2 * sms * 2 * kPartFloats<128> + (size_t)sms * sizeof(JoinTile) / sizeof(float);
}

void launch_attn_tile(const AttnArgs &a, bool e4m3, int sms) {
    if (a.kv.dim == 64) launch_dim<64>(a, e4m3, sms);
    else if (a.kv.dim == 128) launch_dim<128>(a, e4m3, sms);
    else launch_dim<256>(a, e4m3, sms);
}

}  // namespace tq
