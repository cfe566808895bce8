// lora.cu — low-rank adapters of many requests beside a shared projection (x_lora_add).
//
//   y[t] = base[t] + scale[a] (x[t] A[a]^T) B[a]^T,  a = adapter[t];  y[t] = base[t] without one
//
// in two launches for up to four projections that share x: "shrink" h = x A^T (rank values a token)
// and "expand" y = base + h B^T. Both work on tiles of tokens of ONE adapter (64 in shrink, 32 in
// expand), whatever places the tokens have in the batch, so an adapter is read once per 32 or 64 of its
// tokens and never for the others. Each CTA sorts the batch's adapter numbers into tiles itself (at most
// 4096 of a call's tokens at a time): a microsecond for a decode batch, 5 us for 4096 tokens, and it
// spares a launch.
//
// Bytes bound both: x and the adapters in shrink, base, y and the adapters in expand; 2 rank
// operations a value of x or y are below that. x and h are fp32 and enter the bf16 tensor core
// as three bf16 terms, all 24 bits of them: exact up to the fp32 sums, which the tensor core cuts off
// instead of rounding. Shrink moves them to ordinary fp32 sums every 128 values; expand has a sum per term,
// of 256 ranks at most. Operands of one sign, K 5120 to 17408, rank 64: off by 2e-6 of the result. The
// order of shrink's sums follows the tiles that the batch makes (slices, parts of K), so a row's last bits
// depend on the batch that it is in. The
// dimension that is summed is read in the order that suits the loads: a lane takes 16 bytes (8
// neighbouring values) of a row, its share of two k16 steps, the same on both sides.
//
// Measured: 1000 tokens, K 17408, rank 32, 5120 rows: 50 us (shrink 29), where the bytes take 17.6: splitting x
// and the products bound shrink. 4096 tokens, K 5120, rank 64, 10240 rows: 140 us, of which expand moves
// 335 MB in 93. 64 tokens of 24 adapters, 2 x 17408 rows: 46 us (shrink 13); one token: 10 us.
#include "kv.cuh"
#include "tc.cuh"

#include <algorithm>

namespace tq {

namespace {

constexpr int kW = 8;                 // warps of a CTA
constexpr int kTok = 64;              // tokens of a tile of the shrink kernel
constexpr int kTokE = 32;             // and of the expand kernel
constexpr int kMaxTokens = 4096;      // of a launch
constexpr size_t kSmemMost = 232448 - 1024;   // dynamic shared memory of a CTA, beside some static
constexpr int kMaxRank = 256;
constexpr int kMaxSplits = 16;        // parts of K

struct LoraArgs {
    const uint16_t *a[4], *b[4];
    const int *rank[4];
    const float *scale[4];
    const float *base[4];
    float *y[4];
    int M[4], R[4];
    int hoff[5];                      // first column of projection i in a token's row of h
    int count, adapters, K, T;
    const float *x;
    const int *adapter;
    float *h;                         // [splits][T][hoff[count]]
    int max_splits, sms;              // parts of K at most, SMs: see Plan::splits
    int *status;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// ---- the batch's tokens by adapter -------------------------------------------------------------
__device__ __forceinline__ int rank_of(const LoraArgs &a, int i, int id) {
    if (!a.rank[i]) return a.R[i];
    const int r = __ldg(a.rank[i] + id);
    if (r < 0 || r > a.R[i]) atomicCAS(a.status, 0, kStatusAdapter);
    return r < 0 || r > a.R[i] ? 0 : r;
}

// The batch's tokens as tiles of TOK: group 0 is "none", group id + 1 adapter id; s_off[g] = first tile
// of group g, s_id = the groups of the tokens, s_list = the tokens of the tile at hand, in ascending order,
// so that every CTA sees the same tiles.
template <int TOK>
struct Plan {
    int *s_off, *s_cnt, *s_list, *s_sum, *s_tiles;
    uint16_t *s_id;
    __device__ Plan(const LoraArgs &a, uint8_t *smem) {
        s_list = reinterpret_cast<int *>(smem);
        s_sum = s_list + TOK;
        s_tiles = s_sum + kW;
        s_off = s_tiles + 1;
        s_cnt = s_off + a.adapters + 2;
        s_id = reinterpret_cast<uint16_t *>(s_cnt + a.adapters + 1);
    }
    static size_t bytes(int adapters, int T) { return ((size_t)TOK + kW + 2 * adapters + 4) * 4 + ((size_t)T + 1) / 2 * 4; }
    __device__ int tokens(int g, int tile) const { return min(TOK, s_cnt[g] - (tile - s_off[g]) * TOK); }

    // Parts that K is cut into, the same in both kernels: as many as make one round of CTAs of the shrink kernel's
    // tasks. A task's fixed cost (its tokens, its rank, filling the rings, adding the warps' sums) is several us.
    __device__ int splits(const LoraArgs &a) const { return max(1, min(a.max_splits, a.sms / max(1, *s_tiles * a.count))); }

    // All threads of the CTA, of which the first kW warps work. Loops are kept short: code that runs once per launch
    // is fetched from far away, and unrolled it costs more than it saves.
    __device__ void make(const LoraArgs &a) const {
        const int groups = a.adapters + 1, lane = threadIdx.x & 31;
        for (int g = threadIdx.x; g < groups; g += blockDim.x) s_cnt[g] = 0;
        __syncthreads();
        if (threadIdx.x < kW * 32) {
#pragma unroll 1
            for (int t0 = threadIdx.x; t0 - lane < a.T; t0 += 4 * kW * 32) {
                int id[4];                           // loads under way together
#pragma unroll
                for (int i = 0; i < 4; ++i) id[i] = t0 + i * kW * 32 < a.T ? __ldg(a.adapter + t0 + i * kW * 32) : -1;
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                    const int t = t0 + i * kW * 32, v = id[0];
                    id[0] = id[1];
                    id[1] = id[2];
                    id[2] = id[3];
                    if (t - lane >= a.T) break;
                    if (v >= a.adapters) atomicCAS(a.status, 0, kStatusAdapter);
                    // 0 for anything outside the pool, -1 behind the last token
                    const int g = t >= a.T ? -1 : (v >= 0 && v < a.adapters ? v + 1 : 0);
                    if (g >= 0) s_id[t] = (uint16_t)g;
                    // tokens of a request follow one another: the first of a run adds the run
                    const int before = __shfl_up_sync(0xffffffffu, g, 1);
                    const unsigned heads = __ballot_sync(0xffffffffu, lane == 0 || before != g), behind = heads & ~((2u << lane) - 1);
                    if ((heads >> lane & 1) && g >= 0) atomicAdd(s_cnt + g, (behind ? __ffs(behind) - 1 : 32) - lane);
                }
            }
        }
        __syncthreads();
        if (threadIdx.x < 32) {                      // exclusive scan of the groups' tiles
            int tiles = 0, tiles_shrink = 0;
#pragma unroll 1
            for (int g0 = 0; g0 <= groups; g0 += 32) {
                const int g = g0 + lane, m = g < groups ? (s_cnt[g] + TOK - 1) / TOK : 0;
                if (g >= 1 && g < groups) tiles_shrink += (s_cnt[g] + kTok - 1) / kTok;
                int sum = m;
#pragma unroll 1
                for (int off = 1; off < 32; off <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, sum, off);
                    if (lane >= off) sum += o;
                }
                if (g <= groups) s_off[g] = tiles + sum - m;
                tiles += __shfl_sync(0xffffffffu, sum, 31);
            }
            tiles_shrink = __reduce_add_sync(0xffffffffu, tiles_shrink);
            if (lane == 0) *s_tiles = tiles_shrink;
        }
        __syncthreads();
    }
    // The tokens of a tile into s_list; all threads of the CTA, the first kW warps over an eighth of the batch each.
    __device__ void list(const LoraArgs &a, int g, int tile) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, skip = (tile - s_off[g]) * TOK;
        const int chunks = (a.T + kW * 32 - 1) / (kW * 32);      // of 32 tokens, of a warp
        const int t0 = warp * chunks * 32 + lane, t1 = warp < kW ? min(a.T + 31, t0 - lane + chunks * 32) : 0;
        int n = 0;
#pragma unroll 2
        for (int t = t0; t - lane < t1; t += 32) n += __popc(__ballot_sync(0xffffffffu, t < a.T && s_id[t] == g));
        __syncthreads();                             // the list and the sums are no longer read
        if (warp < kW && lane == 0) s_sum[warp] = n;
        __syncthreads();
        int at = -skip;
        for (int w = 0; w < min(warp, kW); ++w) at += s_sum[w];
#pragma unroll 2
        for (int t = t0; t - lane < t1 && at < TOK; t += 32) {
            const bool hit = t < a.T && s_id[t] == g;
            const unsigned votes = __ballot_sync(0xffffffffu, hit);
            const int place = at + __popc(votes & ((1u << lane) - 1));
            if (hit && place >= 0 && place < TOK) s_list[place] = t;
            at += __popc(votes);
        }
        __syncthreads();
    }
};
// The group of tile x: the last g with s_off[g] <= x.
template <int TOK>
__device__ __forceinline__ int group_of(const LoraArgs &a, const Plan<TOK> &p, int x) {
    int lo = 0, hi = a.adapters + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.s_off[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- shrink ------------------------------------------------------------------------------------
// A task is (tile, projection, part of K). Its warps are shared out over the tile's 1 to 4 groups
// of 16 tokens and, for each, slices of the part, whose sums are added through shared memory. The warps
// of a slice bring 64 values of K at a time, each of its 16 rows of x and all together of 64 ranks of A,
// through a ring of theirs (cp.async, 2 to 4 stages; one barrier of theirs a step). Slices take turns at
// the 64 values, so that the CTA reads its rows in runs of 512 bytes or more.
// NB groups of 8 ranks per pass, W warps. The products of 64 ranks keep the tensor cores of mma.sync busy with eight
// warps and their sums fill the registers; up to 32 ranks sixteen warps fit, and they hide more of the latency of
// splitting x: 16, 64, 128 and 1000 tokens of 5 adapters of rank 32, K 17408, take 22.0, 23.6, 32.2 and 50 us with
// sixteen, 20.3, 22.0, 41.0 and 59 us with eight, which therefore serve decode batches (up to 64 tokens).
constexpr int kXBytes = 16 * 256;
constexpr int kRingBytes = 196608;    // of the CTA

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cp_async16_live(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <int NB, int W>
__global__ void __launch_bounds__(W * 32, 1) lora_shrink_kernel(const LoraArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kABytes = NB * 8 * 128;
    static_assert(kRingBytes / 8 >= 2 * (W / 8 * kXBytes + kABytes) && kRingBytes / W >= 16 * (NB * 8 + 2) * 4, "");
    auto sums = [&](int w) { return reinterpret_cast<float (*)[NB * 8 + 2]>(smem + w * (kRingBytes / W)); };   // over the rings
    const Plan<kTok> plan(a, smem + kRingBytes);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    pdl_wait();
    pdl_trigger();
    plan.make(a);
    const int tile0 = plan.s_off[1], tiles = plan.s_off[a.adapters + 1] - tile0;      // group 0 has no product
    const int width = a.hoff[a.count], K64 = (a.K + 63) / 64;
    const int splits = plan.splits(a), per = a.count * splits;
    for (int task = blockIdx.x; task < tiles * per; task += gridDim.x) {
        const int tile = tile0 + task / per, i = task % per / splits, part = task % splits;
        const int g = group_of(a, plan, tile), id = g - 1, tokens = plan.tokens(g, tile);
        if (task == (int)blockIdx.x || tile != tile0 + (task - (int)gridDim.x) / per) plan.list(a, g, tile);
        const int rank = rank_of(a, i, id), R = a.R[i];
        const int k0 = (int)((long long)K64 * part / splits), k1 = (int)((long long)K64 * (part + 1) / splits);
        const int groups16 = (tokens + 15) / 16, slices = min(8, groups16 == 1 ? W : (groups16 == 2 ? W / 2 : W / 4));
        const int team = W / slices, slice = warp / team, m = warp % team;    // m >= groups16: nothing to multiply (three groups)
        const int steps = (k1 - k0 - slice + slices - 1) / slices;
        const int stage_bytes = team * kXBytes + kABytes, stages = kRingBytes / slices / stage_bytes;      // 2, 3 or 4
        const uint32_t ring = smem_u32(smem) + slice * (kRingBytes / slices);
        // this lane's chunks of x: rows 2 c + lane / 16, 16 bytes lane % 16 of 256
        int xt[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int tok = m * 16 + c * 2 + (lane >> 4);
            xt[c] = tok < tokens ? plan.s_list[tok] : -1;
        }
        for (int r0 = 0; r0 < rank; r0 += NB * 8) {
            const int nb = min(NB, (rank - r0 + 7) / 8);
            const uint16_t *A = a.a[i] + ((size_t)id * R + r0) * a.K;
            auto issue = [&](int s) {
                if (s < steps) {
                    const uint32_t dst = ring + s % stages * stage_bytes;
                    const int k = (k0 + slice + s * slices) * 64;
                    // K is a multiple of 32: the last 64 values may be 32
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int r = c * 2 + (lane >> 4), ch = lane & 15;
                        const bool live = xt[c] >= 0 && k + ch * 4 < a.K;
                        cp_async16_live(dst + kABytes + m * kXBytes + r * 256 + ((ch ^ (r & 1)) << 4), live ? a.x + (size_t)xt[c] * a.K + k + ch * 4 : a.x, live);
                    }
#pragma unroll 4
                    for (int n = m; n < nb * 2; n += team) {
                        const int r = n * 4 + (lane >> 3), ch = lane & 7;
                        const bool live = r0 + r < rank && k + ch * 8 < a.K;
                        cp_async16_live(dst + r * 128 + ((ch ^ (r & 1) << 2) << 4), live ? A + (size_t)r * a.K + k + ch * 8 : A, live);
                    }
                }
                cp_async_commit();
            };
            for (int s = 0; s < stages - 1; ++s) issue(s);
            float acc[NB][4], sum[NB][4];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] = sum[n][e] = 0.0f;
            for (int s = 0; s < steps; ++s) {
                // stage s has landed when all but the stages - 2 copies behind it have
                if (stages == 2) cp_async_wait<0>();
                else if (stages == 3) cp_async_wait<1>();
                else cp_async_wait<2>();
                named_bar_sync(1 + slice, team * 32);     // for all warps of the team, which have read stage s - 1
                issue(s + stages - 1);
                if (m >= groups16) continue;
                const uint32_t src = ring + s % stages * stage_bytes, xs = src + kABytes + m * kXBytes;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t f[2][3][4];                  // [k16 step][term]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {         // rows row and row + 8
                        const int r = row + 8 * h;
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint4 v = lds16(xs + r * 256 + (((half * 8 + quad * 2 + z) ^ (r & 1)) << 4));
                            split3(__uint_as_float(v.x), __uint_as_float(v.y), f[z][0][h], f[z][1][h], f[z][2][h]);
                            split3(__uint_as_float(v.z), __uint_as_float(v.w), f[z][0][2 + h], f[z][1][2 + h], f[z][2][2 + h]);
                        }
                    }
                    uint4 w[NB];
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const int r = n * 8 + row;
                        if (n < nb) w[n] = lds16(src + r * 128 + (((half * 4 + quad) ^ (r & 1) << 2) << 4));
                    }
                    // neighbouring products go to different sums: one that needs the last one's waits for it
#pragma unroll
                    for (int z = 0; z < 3; ++z) {
#pragma unroll
                        for (int n = 0; n < NB; ++n)
                            if (n < nb) mma_bf16(acc[n], f[0][z], w[n].x, w[n].y);
#pragma unroll
                        for (int n = 0; n < NB; ++n)
                            if (n < nb) mma_bf16(acc[n], f[1][z], w[n].z, w[n].w);
                    }
                }
                if ((s & 1) || s + 1 == steps) {
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sum[n][e] += acc[n][e];
                            acc[n][e] = 0.0f;
                        }
                }
            }
            cp_async_wait<0>();
            __syncthreads();                              // the rings are free
#pragma unroll
            for (int n = 0; n < NB; ++n)
                if (n < nb) {
                    *reinterpret_cast<float2 *>(&sums(warp)[row][n * 8 + quad * 2]) = make_float2(sum[n][0], sum[n][1]);
                    *reinterpret_cast<float2 *>(&sums(warp)[row + 8][n * 8 + quad * 2]) = make_float2(sum[n][2], sum[n][3]);
                }
            __syncthreads();
            for (int e = threadIdx.x; e < tokens * nb * 8; e += W * 32) {
                const int i_tok = e / (nb * 8), r = e % (nb * 8), t = plan.s_list[i_tok];
                float s = 0.0f;
                for (int w = 0; w < slices; ++w) s += sums(w * team + (i_tok >> 4))[i_tok & 15][r];
                a.h[((size_t)part * a.T + t) * width + a.hoff[i] + r0 + r] = s;
            }
            __syncthreads();
        }
    }
}

// ---- expand ------------------------------------------------------------------------------------
// A task is (tile of 32 tokens, projection, 128 columns of y). The product is taken with the columns as
// the tensor core's rows, D[128 columns][tokens] = B[128][ranks] h^T, so that a warp of the epilogue holds
// 32 neighbouring columns of one token in its lanes: base and y are read and written in whole lines, and
// per token a thread has one load, one addition and one store. (The same product on mma.sync took about
// 1000 clocks a warp for every 16 x 16 results, twice what the memory needed.)
//   load      one thread: 64 ranks of a task's rows of B by TMA into a ring of 16 KB stages, eight ahead
//   mma       one thread: 4 products per 64 ranks, h's three terms beside one another as columns
//   fix       for a rank that ends inside 16: zeros over what lies beyond it in the last product (whatever B holds
//             there must not get in). About a microsecond a task, mostly latency: four warps take tasks in turn
//   epilogue  three teams of four warps, which take turns at the tasks: a team's base rows are under way before it
//             waits for the product, and the other teams' meanwhile
// h of the tile, scaled and split into its terms, lies in shared memory as [64 ranks][term][token], rows of
// 128 bytes with the 128-byte swizzle, as B does. Up to 16 tokens it has 16 rows a term, else 32.
constexpr int kCols = 128;
constexpr int kRing = 8, kBlockB = kCols * 128;
constexpr int kHTile = 3 * kTokE * 128;           // 64 ranks of h, its three terms one below the other
constexpr int kAcc = 4;                           // accumulators in tensor memory, of a column per term and token
constexpr int kAccCols = 128;
constexpr int kFixWarps = 4;
constexpr int kTeams = 3;                         // of four warps, in the epilogue
constexpr int kLoadWarp = 4 * kTeams, kMmaWarp = kLoadWarp + 1, kFixWarp = kMmaWarp + 1;
constexpr int kThreadsE = (kFixWarp + kFixWarps) * 32;

struct LoraMaps {
    CUtensorMap b[4];                             // B as rows [adapter x M] of rank values
};

__device__ __forceinline__ uint32_t idesc_cols(int n) {       // D f32 [128][n], A and B bf16, both K-major
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kCols >> 4) << 24);
}
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {       // K-major rows of 128 bytes, 128-byte swizzle
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}

__global__ void __launch_bounds__(kThreadsE, 1)
    lora_expand_kernel(const LoraArgs a, int chunks_max, unsigned long long limit_ns, const __grid_constant__ LoraMaps maps) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bar[3 * kRing + 2 * kAcc + 1];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u, h_smem = ring + kRing * kBlockB;
    const Plan<kTokE> plan(a, smem_raw + (ring - smem_u32(smem_raw)) + kRing * kBlockB + (size_t)chunks_max * kHTile);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t bars = smem_u32(s_bar);
    auto full = [&](int i) { return bars + 8 * (i & (kRing - 1)); };                     // a stage has landed,
    auto fixed = [&](int i) { return bars + 8 * (kRing + (i & (kRing - 1))); };          // has been mended (counted by themselves),
    auto empty = [&](int i) { return bars + 8 * (2 * kRing + (i & (kRing - 1))); };      // may be written again
    auto acc_full = [&](int i) { return bars + 8 * (3 * kRing + (i & (kAcc - 1))); };
    auto acc_free = [&](int i) { return bars + 8 * (3 * kRing + kAcc + (i & (kAcc - 1))); };
    const uint32_t drained = bars + 8 * (3 * kRing + 2 * kAcc);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 3 * kRing; ++i) mbar_init(bars + 8 * i, 1);
        for (int i = 0; i < kAcc; ++i) {
            mbar_init(acc_full(i), 1);
            mbar_init(acc_free(i), 4);
        }
        mbar_init(drained, 1);
        mbar_init_fence();
        s_gave_up = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&s_tmem), kAcc * kAccCols);
        tmem_relinquish();
        tc_fence_before();
    }
    // The shrink kernel lets this one start behind its own wait for all earlier kernels, so that everything but h
    // may be read from here on.
    plan.make(a);
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int width = a.hoff[a.count], splits = plan.splits(a);
    int blocks = 0;
    bool in_place = true;
    for (int i = 0; i < a.count; ++i) {
        blocks += (a.M[i] + kCols - 1) / kCols;
        in_place = in_place && a.base[i] == a.y[i];
    }
    // the tiles without an adapter come first; in place there is nothing to do for them
    const int tile0 = in_place ? plan.s_off[1] : 0, tiles = plan.s_off[a.adapters + 1] - tile0;
    const int total = tiles * blocks;                // below 2^31 (checked by the entry point)
    const int begin = (int)((long long)total * blockIdx.x / gridDim.x), end = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
    int tile = tile0 + begin / blocks, c = begin % blocks, i = 0, have_tile = -1, g = 0;
    while (c >= (a.M[i] + kCols - 1) / kCols) c -= (a.M[i++] + kCols - 1) / kCols;
    int at = 0, task_no = 0, fixes = 0;              // stages of B so far, tasks with a product, mended stages
    auto hold = [&](uint32_t bar, uint32_t parity) { // by any threads of a warp
        if (mbar_try_wait(bar, parity)) return true;
        if (*(volatile int *)&s_gave_up) return false;
        if (mbar_wait_slow(bar, parity, a.status, 25, limit_ns)) return true;
        *(volatile int *)&s_gave_up = 1;
        return false;
    };
    bool waited = false;
    // runs of tasks of one tile and projection
    for (int task = begin; task < end;) {
        const int n = min(end - task, (a.M[i] + kCols - 1) / kCols - c);
        if (tile != have_tile) g = group_of(a, plan, tile);
        const int id = g - 1, tokens = plan.tokens(g, tile), M = a.M[i];
        const float *base = a.base[i];
        float *const y = a.y[i];
        if (id >= 0 || base != y) {
            if (tile != have_tile) plan.list(a, g, tile);
            else __syncthreads();                    // h and the list are no longer read
            have_tile = tile;
            const int rank = id < 0 ? 0 : rank_of(a, i, id), chunks = (rank + 63) / 64;
            const int fix = rank & 15;               // the last product of the last chunk has ranks that are not the adapter's
            const int blk0 = at, rows_term = tokens > 16 ? 32 : 16;
            auto stage_of = [&](int k, int q) { return blk0 + k * chunks + q; };
            // ---- load: stages [x0, x1) of the run; those of one ring need none of the run's own products
            auto load = [&](int x0, int x1) {
                bool alive = true;
                for (int x = x0; x < x1 && alive; ++x) {
                    const int k = x / chunks, q = x % chunks, st = blk0 + x;
                    if (st >= kRing) alive = hold(empty(st), ((st / kRing) - 1) & 1);
                    if (!alive) break;
                    mbar_expect_tx(full(st), kBlockB);
                    tma_load_2d(ring + (st & (kRing - 1)) * kBlockB, &maps.b[i], q * 64, id * M + (c + k) * kCols, full(st));
                }
            };
            if (warp == kLoadWarp) {
                if (elect_one()) load(0, min(n * chunks, kRing));
                __syncwarp();
            }
            // ---- h of the tile, by all
            if (!waited) {
                pdl_wait();
                pdl_trigger();
                waited = true;
            }
            const float scale = id < 0 ? 0.0f : (a.scale[i] ? __ldg(a.scale[i] + id) : 1.0f);
            for (int e = threadIdx.x; e < chunks * rows_term * 32; e += kThreadsE) {
                const int tok = e >> 5 & (rows_term - 1), q = e / (rows_term * 32), r = q * 64 + (e & 31) * 2;
                float v[2] = {0.0f, 0.0f};
                if (tok < tokens && r < rank) {
                    const float *h = a.h + (size_t)plan.s_list[tok] * width + a.hoff[i] + r;
#pragma unroll 1
                    for (int s0 = 0; s0 < splits; s0 += 8) {
                        float2 part[8];              // all loads under way together
#pragma unroll
                        for (int s = 0; s < 8; ++s)
                            part[s] = s0 + s < splits ? __ldcg(reinterpret_cast<const float2 *>(h + (size_t)(s0 + s) * a.T * width)) : make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int s = 0; s < 8; ++s) {
                            v[0] += part[s].x;
                            v[1] += part[s].y;
                        }
                    }
                }
                v[0] = r < rank ? v[0] * scale : 0.0f;
                v[1] = r + 1 < rank ? v[1] * scale : 0.0f;
                uint32_t t[3];
                split3(v[0], v[1], t[0], t[1], t[2]);
                const uint32_t to = h_smem + q * kHTile + tok * 128 + (((e >> 2 & 7) ^ (tok & 7)) << 4) + (e & 3) * 4;
#pragma unroll
                for (int z = 0; z < 3; ++z) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + z * rows_term * 128), "r"(t[z]) : "memory");
            }
            fence_proxy_async_smem();
            __syncthreads();
            if (warp == kMmaWarp) {
                // ---- mma
                if (elect_one()) {
                    const uint32_t idesc = idesc_cols(3 * rows_term);
                    bool alive = true;
                    for (int k = 0; k < n && chunks && alive; ++k) {
                        const int no = task_no + k;
                        if (no >= kAcc) alive = hold(acc_free(no), ((no / kAcc) - 1) & 1);
                        const uint32_t d = tmem + (no & (kAcc - 1)) * kAccCols;
                        for (int q = 0; q < chunks && alive; ++q) {
                            const int st = stage_of(k, q);
                            alive = fix && q == chunks - 1 ? hold(fixed(fixes + k), ((fixes + k) / kRing) & 1) : hold(full(st), (st / kRing) & 1);
                            if (!alive) break;
                            tc_fence_after();
                            const uint64_t bd = desc_sw128(ring + (st & (kRing - 1)) * kBlockB), hd = desc_sw128(h_smem + q * kHTile);
                            const int steps = min(4, (rank - q * 64 + 15) / 16);
#pragma unroll
                            for (int s = 0; s < 4; ++s)      // 16 ranks are 32 bytes further on
                                if (s < steps) mma_f16_ss(d, bd + 2 * s, hd + 2 * s, idesc, q || s);
                            tc_commit(empty(st));
                        }
                        if (alive) tc_commit(acc_full(no));
                    }
                }
                __syncwarp();                        // the warp comes to the barriers below as one
            } else if (warp == kLoadWarp) {
                if (elect_one()) load(kRing, n * chunks);
                __syncwarp();
            } else if (warp >= kFixWarp) {
                // ---- fix
                bool alive = true;
                for (int k = warp - kFixWarp; k < n && fix && alive; k += kFixWarps) {
                    const int st = stage_of(k, chunks - 1), r0 = (rank & 63) & ~15;      // first rank of the last product, in its chunk
                    alive = __all_sync(0xffffffffu, hold(full(st), (st / kRing) & 1));
                    if (!alive) break;
                    const uint32_t b_smem = ring + (st & (kRing - 1)) * kBlockB;
#pragma unroll 1
                    for (int x = lane; x < kCols * 2; x += 32) {
                        const int m = x >> 1, ch = (r0 >> 3) + (x & 1), keep = fix - (x & 1) * 8;      // values of this chunk that are the adapter's
                        if (keep >= 8) continue;
                        const uint32_t at_m = b_smem + m * 128 + ((ch ^ (m & 7)) << 4);
                        const uint4 v = lds16(at_m);
                        auto word = [&](uint32_t w, int j) { return keep >= 2 * j + 2 ? w : (keep == 2 * j + 1 ? w & 0xffffu : 0u); };
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at_m), "r"(word(v.x, 0)), "r"(word(v.y, 1)), "r"(word(v.z, 2)),
                                     "r"(word(v.w, 3))
                                     : "memory");
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(fixed(fixes + k));
                }
            } else {
                // ---- epilogue
                bool alive = true;
                const int lane_col = (warp & 3) * 32 + lane;
                auto load_base = [&](int k, float (&v)[kTokE]) {
                    const int col = (c + k) * kCols + lane_col;
                    const bool live = base && k < n && col < M;
#pragma unroll
                    for (int t0 = 0; t0 < kTokE; t0 += 8) {
                        if (t0 < tokens) {
#pragma unroll
                            for (int t = t0; t < t0 + 8; ++t) v[t] = live && t < tokens ? base[(size_t)plan.s_list[t] * M + col] : 0.0f;
                        }
                    }
                };
                for (int k = warp >> 2; k < n && alive; k += kTeams) {
                    const int no = task_no + k, col = (c + k) * kCols + lane_col;
                    const bool live = col < M;
                    float v[kTokE];
                    load_base(k, v);
                    if (chunks) {
                        alive = __all_sync(0xffffffffu, hold(acc_full(no), (no / kAcc) & 1));
                        if (!alive) break;
                        tc_fence_after();
                        const uint32_t d = tmem + ((uint32_t)(warp & 3) << 21) + (no & (kAcc - 1)) * kAccCols;
#pragma unroll
                        for (int t0 = 0; t0 < kTokE; t0 += 8) {
                            if (t0 < tokens) {
                                uint32_t w0[8], w1[8], w2[8];
                                tmem_ld8(d + t0, w0);
                                tmem_ld8(d + rows_term + t0, w1);
                                tmem_ld8(d + 2 * rows_term + t0, w2);
                                tmem_wait_ld8(w0);
                                tmem_wait_ld8(w1);
                                tmem_wait_ld8(w2);
#pragma unroll
                                for (int t = 0; t < 8; ++t)
                                    v[t0 + t] += __uint_as_float(w0[t]) + (__uint_as_float(w1[t]) + __uint_as_float(w2[t]));
                            }
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_free(no));
                    }
#pragma unroll
                    for (int t0 = 0; t0 < kTokE; t0 += 8) {
                        if (t0 < tokens) {
#pragma unroll
                            for (int t = t0; t < t0 + 8; ++t)
                                if (live && t < tokens) y[(size_t)plan.s_list[t] * M + col] = v[t];
                        }
                    }
                    __syncwarp();
                }
            }
            at += n * chunks;
            if (chunks) task_no += n;
            if (fix) fixes += n;
        }
        task += n;
        c += n;
        if (c == (M + kCols - 1) / kCols) {
            c = 0;
            if (++i == a.count) {
                i = 0;
                ++tile;
            }
        }
    }
    if (!waited) pdl_wait();
    __syncthreads();
    if (warp == kLoadWarp && s_gave_up && lane == 0)         // copies may still be under way: they end before the CTA does
        for (int st = max(0, at - kRing); st < at; ++st) mbar_wait_bounded(full(st), (st / kRing) & 1, a.status, 25, limit_ns);
    if (warp == kMmaWarp) {
        if (elect_one()) {
            tc_commit(drained);
            mbar_wait_bounded(drained, 0, a.status, 25, limit_ns);
        }
        __syncwarp();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, kAcc * kAccCols);
}

float *g_h = nullptr;
size_t g_h_floats = 0;

}  // namespace
}  // namespace tq

int x_lora_add(const tq_lora_t *const *ws, const float *const *bases, float *const *ys, int count, const float *d_x,
               const int32_t *d_adapter, int T) {
    using namespace tq;
    if (!ws || !ys || count < 1 || count > 4) return -2;
    if (T < 0) return -2;
    LoraArgs a{};
    for (int i = 0; i < count; ++i) {
        const tq_lora_t *w = ws[i];
        if (!w || !w->d_a || !w->d_b || w->count <= 0 || w->rank <= 0 || w->M <= 0 || w->K <= 0) return -1;
        if (w->count != ws[0]->count || w->K != ws[0]->K) return -2;
        if (w->K % 32 || w->M % 16 || w->rank % 8 || w->rank > kMaxRank || w->count > 2048 || w->M > 1 << 21) return -3;
        if ((long long)w->count * w->M > 0x7ffffff0ll) return -3;      // rows of B are counted in 32 bits
        if (!aligned16(w->d_a) || !aligned16(w->d_b)) return -4;
        a.a[i] = w->d_a;
        a.b[i] = w->d_b;
        a.rank[i] = w->d_rank;
        a.scale[i] = w->d_scale;
        a.M[i] = w->M;
        a.R[i] = w->rank;
        a.hoff[i + 1] = a.hoff[i] + w->rank;
    }
    if (!T) return 0;
    if (!d_x || !d_adapter) return -2;
    if (!aligned16(d_x)) return -4;
    for (int i = 0; i < count; ++i) {
        if (!ys[i]) return -2;
        a.base[i] = bases ? bases[i] : nullptr;
        a.y[i] = ys[i];
        if (!aligned16(ys[i]) || (a.base[i] && !aligned16(a.base[i]))) return -4;
    }
    // an output is nobody else's, and x is read for all projections; its own base is the output or apart from it
    const auto bytes = [&](int cols) { return (size_t)T * cols * sizeof(float); };
    for (int i = 0; i < count; ++i) {
        const size_t mine = bytes(a.M[i]);
        if (overlap(ys[i], mine, d_x, bytes(ws[0]->K))) return -2;
        if (ys[i] != a.base[i] && overlap(ys[i], mine, a.base[i], mine)) return -2;
        for (int j = 0; j < count; ++j)
            if (j != i && (overlap(ys[i], mine, ys[j], bytes(a.M[j])) || overlap(ys[i], mine, a.base[j], bytes(a.M[j])))) return -2;
    }
    a.count = count;
    a.adapters = ws[0]->count;
    a.K = ws[0]->K;
    a.T = T;
    a.x = d_x;
    a.adapter = d_adapter;
    const int sms = gpu_sms();
    // a call of more tokens than a CTA sorts goes in pieces
    const int piece = std::min(T, kMaxTokens), k64 = (a.K + 63) / 64;
    const int tiles = (piece + kTok - 1) / kTok + std::min(piece, a.adapters);     // at most
    // A step for every warp at least. The kernels cut K by the tiles that there are (Plan::splits); this is the most.
    a.max_splits = std::max(1, std::min({kMaxSplits, sms / ((piece + kTok - 1) / kTok * count), k64 / kW}));
    a.sms = sms;
    const size_t need = (size_t)a.max_splits * piece * a.hoff[count];
    if (need > g_h_floats) {
        if (stream_is_capturing()) return -40;
        // The last scratch stays allocated: a graph may have been captured with it. Each is twice the last at least.
        g_h_floats = std::max(need, 2 * g_h_floats);
        g_h = static_cast<float *>(tq_dev_alloc(g_h_floats * sizeof(float), "lora.h"));
    }
    a.h = g_h;
    if (!device_status_ready()) return -40;
    a.status = device_status_word();
    int most = 0;
    long long blocks = 0;
    LoraMaps maps{};
    for (int i = 0; i < count; ++i) {
        most = std::max(most, a.R[i]);
        blocks += (a.M[i] + kCols - 1) / kCols;
        if (!tensor_map_2d(maps.b[i], a.b[i], a.R[i], (long long)a.adapters * a.M[i], kCols)) return -3;
    }
    const int tiles_e = (piece + kTokE - 1) / kTokE + std::min(piece, a.adapters + 1);
    if (blocks * tiles_e > 0x7fffffffll) return -3;
    const int chunks = (most + 63) / 64;
    const size_t shrink_smem = (size_t)kRingBytes + Plan<kTok>::bytes(a.adapters, piece);
    const size_t expand_smem = 1024 + (size_t)kRing * kBlockB + (size_t)chunks * kHTile + Plan<kTokE>::bytes(a.adapters, piece);
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(lora_shrink_kernel<4, 16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
        TQ_CHECK(cudaFuncSetAttribute(lora_shrink_kernel<8, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
        TQ_CHECK(cudaFuncSetAttribute(lora_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
        set = true;
    }
    for (int t0 = 0; t0 < T; t0 += kMaxTokens) {
        a.T = std::min(kMaxTokens, T - t0);
        a.x = d_x + (size_t)t0 * a.K;
        a.adapter = d_adapter + t0;
        for (int i = 0; i < count; ++i) {
            a.base[i] = bases && bases[i] ? bases[i] + (size_t)t0 * a.M[i] : nullptr;
            a.y[i] = ys[i] + (size_t)t0 * a.M[i];
        }
        const int shrink = (int)std::min<long long>((long long)tiles * count * a.max_splits, sms);
        const int expand = (int)std::min<long long>(tiles_e * blocks, sms);
        if (most <= 32 && piece > kTok) launch_pdl(lora_shrink_kernel<4, 16>, dim3(shrink), dim3(16 * 32), shrink_smem, a);
        else launch_pdl(lora_shrink_kernel<8, 8>, dim3(shrink), dim3(8 * 32), shrink_smem, a);
        launch_pdl(lora_expand_kernel, dim3(expand), dim3(kThreadsE), expand_smem, a, chunks, wait_limit_ns(), maps);
    }
    TQ_LAUNCH_CHECK("lora_expand_kernel");
    return 0;
}
