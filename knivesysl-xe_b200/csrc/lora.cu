// lora.cu — low-rank adapters of many requests beside a shared projection (x_lora_add).
//
//   y[t] = base[t] + scale[a] (x[t] A[a]^T) B[a]^T,  a = adapter[t];  y[t] = base[t] without one
//
// in two launches for up to four projections that share x: "shrink" h = x A^T (rank values a token)
// and "expand" y = base + h B^T. Both work on tiles of up to 64 tokens of ONE adapter, whatever
// places the tokens have in the batch: 16 of them are the m side of an mma, the adapter's rows the n
// side, so an adapter is read once per 64 of its tokens and never for the others. Each CTA sorts the
// batch's adapter numbers into tiles itself (at most 4096 of a call's tokens at a time), which takes
// it about a microsecond and spares a launch.
//
// Bytes bound both: x and the adapters in shrink, base, y and the adapters in expand; 2 rank
// operations a value of x or y are far below that. x and h are fp32 and enter the bf16 tensor core
// as three bf16 terms, all 24 bits of them: exact up to the fp32 sums, which the tensor core cuts off
// instead of rounding and which are therefore moved to ordinary fp32 sums every 128 values. The
// dimension that is summed is read in the order that suits the loads: a lane takes 16 bytes (8
// neighbouring values) of a row, its share of two k16 steps, the same on both sides.
#include "kv.cuh"
#include "tc.cuh"

#include <algorithm>

namespace tq {

namespace {

constexpr int kW = 8;                 // warps of a CTA
constexpr int kTok = 64;              // tokens of a tile of the shrink kernel
constexpr int kTokE = 32;             // and of the expand kernel
constexpr int kMaxTokens = 4096;      // of a launch
constexpr size_t kSmemMost = 232448 - 256;   // dynamic shared memory of a CTA, beside some static
constexpr int kMaxRank = 256;

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
    int splits;                       // parts of K, summed in ascending order by the expand kernel
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
    int *s_off, *s_cnt, *s_list, *s_sum;
    uint16_t *s_id;
    __device__ Plan(const LoraArgs &a, uint8_t *smem) {
        s_list = reinterpret_cast<int *>(smem);
        s_sum = s_list + TOK;
        s_off = s_sum + kW;
        s_cnt = s_off + a.adapters + 2;
        s_id = reinterpret_cast<uint16_t *>(s_cnt + a.adapters + 1);
    }
    static size_t bytes(int adapters, int T) { return ((size_t)TOK + kW + 2 * adapters + 3) * 4 + ((size_t)T + 1) / 2 * 4; }
    __device__ int tokens(int g, int tile) const { return min(TOK, s_cnt[g] - (tile - s_off[g]) * TOK); }

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
            int tiles = 0;
#pragma unroll 1
            for (int g0 = 0; g0 <= groups; g0 += 32) {
                const int g = g0 + lane, m = g < groups ? (s_cnt[g] + TOK - 1) / TOK : 0;
                int sum = m;
#pragma unroll 1
                for (int off = 1; off < 32; off <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, sum, off);
                    if (lane >= off) sum += o;
                }
                if (g <= groups) s_off[g] = tiles + sum - m;
                tiles += __shfl_sync(0xffffffffu, sum, 31);
            }
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
// A task is (tile, projection, part of K). Its eight warps are shared out over the tile's 1 to 4 groups
// of 16 tokens and, for each, slices of the part, whose sums are added through shared memory. A warp
// brings 64 values of K of its 16 rows of x and of 64 ranks of A at a time through a ring of its own
// (cp.async). Slices take turns at the 64 values, so that the CTA reads its rows in runs of 512 bytes or more.
constexpr int kNB = 8;                // groups of 8 ranks per pass
constexpr int kStages = 2;
constexpr int kXBytes = 16 * 256, kABytes = kNB * 8 * 128, kStageBytes = kXBytes + kABytes;

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cp_async16_live(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// through L1, for what other warps of the CTA read at about the same time
__device__ __forceinline__ void cp_async16_shared(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__global__ void __launch_bounds__(kW * 32, 1) lora_shrink_kernel(const LoraArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    auto sums = [&](int w) { return reinterpret_cast<float (*)[kNB * 8 + 2]>(smem + w * kStages * kStageBytes); };   // over the rings
    const Plan<kTok> plan(a, smem + kW * kStages * kStageBytes);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
    pdl_wait();
    pdl_trigger();
    plan.make(a);
    const int tile0 = plan.s_off[1], tiles = plan.s_off[a.adapters + 1] - tile0;      // group 0 has no product
    const int width = a.hoff[a.count], K64 = (a.K + 63) / 64;
    const int per = a.count * a.splits;
    for (int task = blockIdx.x; task < tiles * per; task += gridDim.x) {
        const int tile = tile0 + task / per, i = task % per / a.splits, part = task % a.splits;
        const int g = group_of(a, plan, tile), id = g - 1, tokens = plan.tokens(g, tile);
        if (task == (int)blockIdx.x || tile != tile0 + (task - (int)gridDim.x) / per) plan.list(a, g, tile);
        const int rank = rank_of(a, i, id), R = a.R[i];
        const int k0 = (int)((long long)K64 * part / a.splits), k1 = (int)((long long)K64 * (part + 1) / a.splits);
        const int groups16 = (tokens + 15) / 16, slices = groups16 == 1 ? 8 : (groups16 == 2 ? 4 : 2);
        const int m = warp / slices, slice = warp % slices;    // m >= groups16: nothing to do (three groups)
        const int steps = m < groups16 ? (k1 - k0 - slice + slices - 1) / slices : 0;
        // this lane's chunks of x: rows 2 c + lane / 16, 16 bytes lane % 16 of 256
        int xt[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int tok = m * 16 + c * 2 + (lane >> 4);
            xt[c] = tok < tokens ? plan.s_list[tok] : -1;
        }
        for (int r0 = 0; r0 < rank; r0 += kNB * 8) {
            const int nb = min(kNB, (rank - r0 + 7) / 8);
            const uint16_t *A = a.a[i] + ((size_t)id * R + r0) * a.K;
            auto issue = [&](int s) {
                if (s < steps) {
                    const uint32_t dst = ring + s % kStages * kStageBytes;
                    const int k = (k0 + slice + s * slices) * 64;
                    // K is a multiple of 32: the last 64 values may be 32
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int r = c * 2 + (lane >> 4), ch = lane & 15;
                        const bool live = xt[c] >= 0 && k + ch * 4 < a.K;
                        cp_async16_live(dst + r * 256 + ((ch ^ (r & 1)) << 4), live ? a.x + (size_t)xt[c] * a.K + k + ch * 4 : a.x, live);
                    }
#pragma unroll
                    for (int n = 0; n < kNB * 2; ++n)
                        if (n < nb * 2) {
                            const int r = n * 4 + (lane >> 3), ch = lane & 7;
                            const bool live = r0 + r < rank && k + ch * 8 < a.K;
                            cp_async16_shared(dst + kXBytes + r * 128 + ((ch ^ (r & 1) << 2) << 4), live ? A + (size_t)r * a.K + k + ch * 8 : A, live);
                        }
                }
                cp_async_commit();
            };
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) issue(s);
            float acc[kNB][4], sum[kNB][4];
#pragma unroll
            for (int n = 0; n < kNB; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] = sum[n][e] = 0.0f;
            for (int s = 0; s < steps; ++s) {
                issue(s + kStages - 1);
                cp_async_wait<kStages - 1>();
                __syncwarp();
                const uint32_t src = ring + s % kStages * kStageBytes;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t f[2][3][4];                  // [k16 step][term]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {         // rows row and row + 8
                        const int r = row + 8 * h;
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint4 v = lds16(src + r * 256 + (((half * 8 + quad * 2 + z) ^ (r & 1)) << 4));
                            split3(__uint_as_float(v.x), __uint_as_float(v.y), f[z][0][h], f[z][1][h], f[z][2][h]);
                            split3(__uint_as_float(v.z), __uint_as_float(v.w), f[z][0][2 + h], f[z][1][2 + h], f[z][2][2 + h]);
                        }
                    }
                    uint4 w[kNB];
#pragma unroll
                    for (int n = 0; n < kNB; ++n) {
                        const int r = n * 8 + row;
                        if (n < nb) w[n] = lds16(src + kXBytes + r * 128 + (((half * 4 + quad) ^ (r & 1) << 2) << 4));
                    }
                    // neighbouring products go to different sums: one that needs the last one's waits for it
#pragma unroll
                    for (int z = 0; z < 3; ++z) {
#pragma unroll
                        for (int n = 0; n < kNB; ++n)
                            if (n < nb) mma_bf16(acc[n], f[0][z], w[n].x, w[n].y);
#pragma unroll
                        for (int n = 0; n < kNB; ++n)
                            if (n < nb) mma_bf16(acc[n], f[1][z], w[n].z, w[n].w);
                    }
                }
                if ((s & 1) || s + 1 == steps) {
#pragma unroll
                    for (int n = 0; n < kNB; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            sum[n][e] += acc[n][e];
                            acc[n][e] = 0.0f;
                        }
                }
                __syncwarp();                             // all lanes have read the stage
            }
            cp_async_wait<0>();
            __syncwarp();
#pragma unroll
            for (int n = 0; n < kNB; ++n)
                if (n < nb) {
                    *reinterpret_cast<float2 *>(&sums(warp)[row][n * 8 + quad * 2]) = make_float2(sum[n][0], sum[n][1]);
                    *reinterpret_cast<float2 *>(&sums(warp)[row + 8][n * 8 + quad * 2]) = make_float2(sum[n][2], sum[n][3]);
                }
            __syncthreads();
            for (int e = threadIdx.x; e < tokens * nb * 8; e += kW * 32) {
                const int i_tok = e / (nb * 8), r = e % (nb * 8), t = plan.s_list[i_tok];
                float s = 0.0f;
                for (int w = 0; w < slices; ++w) s += sums((i_tok >> 4) * slices + w)[i_tok & 15][r];
                a.h[((size_t)part * a.T + t) * width + a.hoff[i] + r0 + r] = s;
            }
            __syncthreads();
        }
    }
}

// The first n of 8 values, zeros behind them.
__device__ __forceinline__ uint4 first_values(uint4 v, int n) {
    auto word = [&](uint32_t x, int i) { return n >= 2 * i + 2 ? x : (n == 2 * i + 1 ? x & 0xffffu : 0u); };
    return make_uint4(word(v.x, 0), word(v.y, 1), word(v.z, 2), word(v.w, 3));
}

// ---- expand ------------------------------------------------------------------------------------
// A task is (tile of 32 tokens, projection, block of columns): 256 columns with up to 64 ranks, 128 or
// 64 with more, so that a block of B, which is one piece of memory, has at most 32 KB. A warp of its own
// brings the block of B and the tokens' base rows (1 KB each) into a stage of shared memory by bulk
// copies, up to three tasks ahead; the sixteen others multiply 32 columns by 16 tokens each, add and
// store. So 130 KB an SM are under way whatever the products do. h of the tile, scaled and split into its terms, lies in shared memory
// as [term][token][rank].
constexpr int kWE = 16;                           // warps that multiply
constexpr int kThreadsE = kWE * 32 + 32;
constexpr int kRowPitch = 1024 + 64;              // bytes of a token's row in a stage: rows of 8 lanes on different banks
constexpr int kBBytes = 32768;
constexpr int kTaskBytes = kTokE * kRowPitch + kBBytes;
__host__ __device__ inline int task_cols(int R) { return R <= 64 ? 256 : (R <= 128 ? 128 : 64); }
__host__ __device__ inline int task_blocks(int M, int R) { return (M + task_cols(R) - 1) / task_cols(R); }
// The column that row `row` of a warp's n8 tile n stands for: a lane's results in tiles 2i and 2i + 1 are
// four neighbouring columns.
__device__ __forceinline__ int column(int n, int row) { return (n >> 1) * 16 + (row >> 1) * 4 + (n & 1) * 2 + (row & 1); }
__global__ void __launch_bounds__(kThreadsE, 1) lora_expand_kernel(const LoraArgs a, int pitch, int stages, unsigned long long limit_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_bar[6];
    __shared__ int s_gave_up;
    // pitch: ranks rounded up to 32, and 8 more: the rows of 8 lanes lie on different banks
    uint16_t *const s_h = reinterpret_cast<uint16_t *>(smem + stages * kTaskBytes);
    const int plane = kTokE * pitch;
    const Plan<kTokE> plan(a, reinterpret_cast<uint8_t *>(s_h + 3 * plane));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    const uint32_t stage0 = smem_u32(smem), bars = smem_u32(s_bar);
    auto full = [&](int s) { return bars + 8 * s; };             // a stage holds its task's operands
    auto done = [&](int s) { return bars + 8 * (3 + s); };       // and they have been read
    if (threadIdx.x == 0) {
        for (int s = 0; s < 3; ++s) {
            mbar_init(full(s), 1);
            mbar_init(done(s), kWE);
        }
        mbar_init_fence();
        s_gave_up = 0;
    }
    pdl_wait();
    pdl_trigger();
    plan.make(a);
    const int tiles = plan.s_off[a.adapters + 1], width = a.hoff[a.count];
    int blocks = 0;
    for (int i = 0; i < a.count; ++i) blocks += task_blocks(a.M[i], a.R[i]);
    const int total = tiles * blocks;                // below 2^31 (checked by the entry point)
    const int begin = (int)((long long)total * blockIdx.x / gridDim.x), end = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
    int tile = begin / max(1, blocks), c = begin % max(1, blocks), i = 0, have_tile = -1, g = 0;
    while (c >= task_blocks(a.M[i], a.R[i])) c -= task_blocks(a.M[i], a.R[i++]);
    int at = 0, loaded = 0;                          // tasks so far (stage at % stages), and those begun to load
    bool alive = true;
    auto hold = [&](uint32_t bar, uint32_t parity) { // by a whole warp
        if (mbar_test_wait_warp(bar, parity)) return true;
        bool ok = false;
        if (!*(volatile int *)&s_gave_up) {
            ok = mbar_wait_slow(bar, parity, a.status, 25, limit_ns);
            if (!ok) *(volatile int *)&s_gave_up = 1;
        }
        return (bool)__all_sync(0xffffffffu, ok);
    };
    // runs of tasks of one tile and projection
    for (int task = begin; task < end;) {
        const int cols = task_cols(a.R[i]), n = min(end - task, task_blocks(a.M[i], a.R[i]) - c);
        if (tile != have_tile) g = group_of(a, plan, tile);
        const int id = g - 1, tokens = plan.tokens(g, tile), R = a.R[i], M = a.M[i];
        const float *base = a.base[i];
        float *const y = a.y[i];
        if (id >= 0 || base != y) {
            if (tile != have_tile) plan.list(a, g, tile);
            else __syncthreads();                    // h is no longer read
            have_tile = tile;
            const int rank = id < 0 ? 0 : rank_of(a, i, id);
            const uint16_t *B = a.b[i] + (size_t)max(id, 0) * M * R;
            auto load = [&](int k) {                 // operands of the run's task k (warp kWE)
                const int s = (at + k) % stages, col0 = (c + k) * cols, w = min(cols, M - col0);
                const uint32_t dst = stage0 + s * kTaskBytes;
                loaded = at + k + 1;
                if (lane == 0) mbar_expect_tx(full(s), (base ? tokens * w * 4 : 0) + (rank ? w * R * 2 : 0));
                __syncwarp();
                if (rank && lane == 0) bulk_g2s_plain(dst + kTokE * kRowPitch, B + (size_t)col0 * R, w * R * 2, full(s));
                if (base && lane < tokens) bulk_g2s_plain(dst + lane * kRowPitch, base + (size_t)plan.s_list[lane] * M + col0, w * 4, full(s));
            };
            if (warp == kWE)
                for (int k = 0; k < min(stages, n) && alive; ++k) load(k);
            // h of the tile
            const int pad = (rank + 31) & ~31, rows16 = (tokens + 15) & ~15;
            const float scale = id < 0 ? 0.0f : (a.scale[i] ? __ldg(a.scale[i] + id) : 1.0f);
            for (int e = threadIdx.x; e < rows16 * (pad / 2); e += kThreadsE) {
                const int i_tok = e / (pad / 2), r = e % (pad / 2) * 2;
                float v[2] = {0.0f, 0.0f};
                if (i_tok < tokens && r < rank) {
                    const float *h = a.h + (size_t)plan.s_list[i_tok] * width + a.hoff[i] + r;
                    float2 part[8];                  // at most 8 parts, all loads under way together
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        part[s] = s < a.splits ? __ldcg(reinterpret_cast<const float2 *>(h + (size_t)s * a.T * width)) : make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        v[0] += part[s].x;
                        v[1] += part[s].y;
                    }
                }
                v[0] = r < rank ? v[0] * scale : 0.0f;
                v[1] = r + 1 < rank ? v[1] * scale : 0.0f;
                uint32_t t0, t1, t2;
                split3(v[0], v[1], t0, t1, t2);
                uint32_t *dst = reinterpret_cast<uint32_t *>(s_h + i_tok * pitch + r);
                dst[0] = t0;
                dst[plane / 2] = t1;
                dst[plane] = t2;
            }
            __syncthreads();
            if (warp == kWE) {
                for (int k = 0; k < n && alive; ++k) {
                    const int s = (at + k) % stages;
                    alive = hold(done(s), ((at + k) / stages) & 1);
                    if (alive && k + stages < n) load(k + stages);
                }
            } else {
                const int across = cols / 32, wc = warp % across * 32, w16 = warp / across, step16 = kWE / across;
                const bool odd = rank & 7;           // a rank that ends inside a lane's 16 bytes
                for (int k = 0; k < n && alive; ++k) {
                    const int s = (at + k) % stages, w = min(cols, M - (c + k) * cols);
                    const uint8_t *const rows = smem + s * kTaskBytes;
                    const uint8_t *const bs = rows + kTokE * kRowPitch;
                    alive = hold(full(s), ((at + k) / stages) & 1);
                    if (!alive) break;
                    for (int m16 = w16; m16 * 16 < tokens; m16 += step16) {
                        float acc[4][4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.0f;
                        for (int r0 = 0; r0 < rank; r0 += 32) {
                            uint4 b[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int m = wc + column(q, row), r = r0 + quad * 8;
                                b[q] = m < w && r < rank ? *reinterpret_cast<const uint4 *>(bs + ((size_t)m * R + r) * 2) : make_uint4(0, 0, 0, 0);
                                if (odd && r + 8 > rank) b[q] = first_values(b[q], rank - r);
                            }
#pragma unroll
                            for (int z = 0; z < 3; ++z) {
                                const uint16_t *hp = s_h + z * plane + (m16 * 16 + row) * pitch + r0 + quad * 8;
                                const uint4 lo = *reinterpret_cast<const uint4 *>(hp), hi = *reinterpret_cast<const uint4 *>(hp + 8 * pitch);
                                const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q) mma_bf16(acc[q], f0, b[q].x, b[q].y);
#pragma unroll
                                for (int q = 0; q < 4; ++q) mma_bf16(acc[q], f1, b[q].z, b[q].w);
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int tok = m16 * 16 + row + 8 * h;
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const int col = wc + q * 16 + quad * 4;
                                if (tok >= tokens || col >= w) continue;
                                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (base) v = *reinterpret_cast<const float4 *>(rows + tok * kRowPitch + col * 4);
                                v.x += acc[2 * q][2 * h];
                                v.y += acc[2 * q][2 * h + 1];
                                v.z += acc[2 * q + 1][2 * h];
                                v.w += acc[2 * q + 1][2 * h + 1];
                                *reinterpret_cast<float4 *>(y + (size_t)plan.s_list[tok] * M + (c + k) * cols + col) = v;
                            }
                        }
                    }
                    __syncwarp();                    // all lanes have read the stage
                    if (lane == 0) mbar_arrive(done(s));
                }
            }
            at += n;
        }
        task += n;
        c += n;
        if (c == task_blocks(M, R)) {
            c = 0;
            if (++i == a.count) {
                i = 0;
                ++tile;
            }
        }
        if (*(volatile int *)&s_gave_up) alive = false;
    }
    if (warp == kWE) {
        if (!alive)                                  // a wait gave up: the copies under way end before the CTA does
            for (int k = max(0, loaded - stages); k < loaded; ++k)
                mbar_wait_bounded(full(k % stages), (k / stages) & 1, a.status, 25, limit_ns);
    }
}

float *g_h = nullptr;
size_t g_h_floats = 0;

int sm_count() {
    static int n = 0;
    if (!n) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, tq_device());
    return n > 0 ? n : 148;
}

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
    a.count = count;
    a.adapters = ws[0]->count;
    a.K = ws[0]->K;
    a.T = T;
    a.x = d_x;
    a.adapter = d_adapter;
    const int sms = sm_count();
    // a call of more tokens than a CTA sorts goes in pieces
    const int piece = std::min(T, kMaxTokens), k64 = (a.K + 63) / 64;
    const int tiles = (piece + kTok - 1) / kTok + std::min(piece, a.adapters);     // at most
    // one round of CTAs: a task's fixed cost (its tokens, its rank, filling the rings, adding the warps' sums) is
    // several us; and a step for every warp at least
    a.splits = std::max(1, std::min({8, sms / std::max(1, tiles * count), k64 / kW}));
    const size_t need = (size_t)a.splits * piece * a.hoff[count];
    if (need > g_h_floats) {
        if (stream_is_capturing()) return -40;
        if (g_h) tq_dev_free(g_h);
        g_h = static_cast<float *>(tq_dev_alloc(need * sizeof(float), "lora.h"));
        g_h_floats = need;
    }
    a.h = g_h;
    if (!device_status_ready()) return -40;
    a.status = device_status_word();
    int most = 0;
    long long blocks = 0;
    for (int i = 0; i < count; ++i) {
        most = std::max(most, a.R[i]);
        blocks += task_blocks(a.M[i], a.R[i]);
    }
    const int tiles_e = (piece + kTokE - 1) / kTokE + std::min(piece, a.adapters + 1);
    if (blocks * tiles_e > 0x7fffffffll) return -3;
    const int pitch = ((most + 31) & ~31) + 8;
    const size_t shrink_smem = (size_t)kW * kStages * kStageBytes + Plan<kTok>::bytes(a.adapters, piece);
    const size_t rest = (size_t)3 * kTokE * pitch * 2 + Plan<kTokE>::bytes(a.adapters, piece);
    const int stages = 3 * kTaskBytes + rest <= kSmemMost ? 3 : 2;
    const size_t expand_smem = stages * kTaskBytes + rest;
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
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
        const int shrink = (int)std::min<long long>((long long)tiles * count * a.splits, sms);
        const int expand = (int)std::min<long long>(tiles_e * blocks, sms);
        launch_pdl(lora_shrink_kernel, dim3(shrink), dim3(kW * 32), shrink_smem, a);
        launch_pdl(lora_expand_kernel, dim3(expand), dim3(kThreadsE), expand_smem, a, pitch, stages, wait_limit_ns());
    }
    TQ_LAUNCH_CHECK("lora_expand_kernel");
    return 0;
}
