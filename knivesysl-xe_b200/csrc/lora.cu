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

#include <algorithm>

namespace tq {

namespace {

constexpr int kW = 8;                 // warps of a CTA
constexpr int kTok = 64;              // tokens of a tile
constexpr int kMaxTokens = 4096;      // of a launch
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
// Adapter numbers as this kernel takes them: -1 (none) for anything outside the pool.
__device__ __forceinline__ int adapter_of(const LoraArgs &a, int t) {
    const int id = __ldg(a.adapter + t);
    if (id >= a.adapters) atomicCAS(a.status, 0, kStatusAdapter);
    return id >= 0 && id < a.adapters ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &a, int i, int id) {
    if (!a.rank[i]) return a.R[i];
    const int r = __ldg(a.rank[i] + id);
    if (r < 0 || r > a.R[i]) atomicCAS(a.status, 0, kStatusAdapter);
    return r < 0 || r > a.R[i] ? 0 : r;
}

// The batch's tokens as tiles: group 0 is "none", group id + 1 adapter id; s_off[g] = first tile of group
// g, s_id = the groups of the tokens, s_list = the tokens of the tile at hand, in ascending order, so
// that every CTA sees the same tiles.
struct Plan {
    int *s_off, *s_cnt, *s_list, *s_sum;
    uint16_t *s_id;
    __device__ Plan(const LoraArgs &a, uint8_t *smem) {
        s_list = reinterpret_cast<int *>(smem);
        s_sum = s_list + kTok;
        s_off = s_sum + kW;
        s_cnt = s_off + a.adapters + 2;
        s_id = reinterpret_cast<uint16_t *>(s_cnt + a.adapters + 1);
    }
    static size_t bytes(int adapters, int T) { return ((size_t)kTok + kW + 2 * adapters + 3) * 4 + ((size_t)T + 1) / 2 * 4; }
    __device__ int tokens(int g, int tile) const { return min(kTok, s_cnt[g] - (tile - s_off[g]) * kTok); }
};
// All threads of the CTA.
__device__ void make_plan(const LoraArgs &a, const Plan &p) {
    const int groups = a.adapters + 1, lane = threadIdx.x & 31;
    for (int g = threadIdx.x; g < groups; g += kW * 32) p.s_cnt[g] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < a.T; t0 += kW * 32) {
        const int t = t0 + threadIdx.x, g = t < a.T ? adapter_of(a, t) + 1 : -1;
        if (g >= 0) p.s_id[t] = (uint16_t)g;
        const unsigned same = __match_any_sync(0xffffffffu, g);
        if (g >= 0 && lane == __ffs(same) - 1) atomicAdd(p.s_cnt + g, __popc(same));
    }
    __syncthreads();
    if (threadIdx.x < 32) {                          // exclusive scan of the groups' tiles
        int tiles = 0;
        for (int g0 = 0; g0 <= groups; g0 += 32) {
            const int g = g0 + lane, m = g < groups ? (p.s_cnt[g] + kTok - 1) / kTok : 0;
            int sum = m;
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, sum, off);
                if (lane >= off) sum += o;
            }
            if (g <= groups) p.s_off[g] = tiles + sum - m;
            tiles += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    __syncthreads();
}
// The tokens of a tile into s_list; all threads of the CTA, each warp over an eighth of the batch.
__device__ void list_tile(const LoraArgs &a, const Plan &p, int g, int tile) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, skip = (tile - p.s_off[g]) * kTok;
    const int span = ((a.T + kW * 32 - 1) / (kW * 32)) * 32, t0 = warp * span, t1 = min(a.T, t0 + span);
    int n = 0;
    for (int t = t0; t < t1; t += 32) n += __popc(__ballot_sync(0xffffffffu, t + lane < t1 && p.s_id[t + lane] == g));
    __syncthreads();                                 // the list and the sums are no longer read
    if (lane == 0) p.s_sum[warp] = n;
    __syncthreads();
    int at = -skip;
    for (int w = 0; w < warp; ++w) at += p.s_sum[w];
    for (int t = t0; t < t1 && at < kTok; t += 32) {
        const bool hit = t + lane < t1 && p.s_id[t + lane] == g;
        const unsigned votes = __ballot_sync(0xffffffffu, hit);
        const int place = at + __popc(votes & ((1u << lane) - 1));
        if (hit && place >= 0 && place < kTok) p.s_list[place] = t + lane;
        at += __popc(votes);
    }
    __syncthreads();
}
// The group of tile x: the last g with s_off[g] <= x.
__device__ __forceinline__ int group_of(const LoraArgs &a, const Plan &p, int x) {
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
    const Plan plan(a, smem + kW * kStages * kStageBytes);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
    pdl_wait();
    pdl_trigger();
    make_plan(a, plan);
    const int tile0 = plan.s_off[1], tiles = plan.s_off[a.adapters + 1] - tile0;      // group 0 has no product
    const int width = a.hoff[a.count], K64 = (a.K + 63) / 64;
    const int per = a.count * a.splits;
    for (int task = blockIdx.x; task < tiles * per; task += gridDim.x) {
        const int tile = tile0 + task / per, i = task % per / a.splits, part = task % a.splits;
        const int g = group_of(a, plan, tile), id = g - 1, tokens = plan.tokens(g, tile);
        if (task == (int)blockIdx.x || tile != tile0 + (task - (int)gridDim.x) / per) list_tile(a, plan, g, tile);
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
// A task is (tile, projection, 256 columns of y): 32 columns a warp, whose rows of B (up to 64 ranks)
// stay in registers while the tile's groups of 16 tokens go by, the next group's base rows under way.
// h of the tile, scaled and split into its terms, lies in shared memory as [term][token][rank].
constexpr int kCols = 32 * kW;
__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// The column that row `row` of a warp's n8 tile n stands for: a lane's results in tiles 2i and 2i + 1 are
// four neighbouring columns.
__device__ __forceinline__ int column(int n, int row) { return (n >> 1) * 16 + (row >> 1) * 4 + (n & 1) * 2 + (row & 1); }

__global__ void __launch_bounds__(kW * 32, 2) lora_expand_kernel(const LoraArgs a, int pitch) {
    extern __shared__ __align__(16) uint8_t smem[];
    // pitch: ranks rounded up to 32, and 8 more: the rows of 8 lanes lie on different banks
    uint16_t *const s_h = reinterpret_cast<uint16_t *>(smem);
    const int plane = kTok * pitch;
    const Plan plan(a, smem + (size_t)3 * plane * 2);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    pdl_wait();
    pdl_trigger();
    make_plan(a, plan);
    const int tiles = plan.s_off[a.adapters + 1], width = a.hoff[a.count];
    int blocks = 0;
    for (int i = 0; i < a.count; ++i) blocks += (a.M[i] + kCols - 1) / kCols;
    const int total = tiles * blocks;                // below 2^31: 2112 tiles at most, of 2^15 blocks (checked by the entry point)
    const int begin = (int)((long long)total * blockIdx.x / gridDim.x), end = (int)((long long)total * (blockIdx.x + 1) / gridDim.x);
    int tile = begin / blocks, c = begin % blocks, i = 0, have_tile = -1, have_i = -1, rank = 0, g = 0;
    while (c >= (a.M[i] + kCols - 1) / kCols) c -= (a.M[i++] + kCols - 1) / kCols;
    for (int task = begin; task < end; ++task, ++c) {
        if (c == (a.M[i] + kCols - 1) / kCols) {
            c = 0;
            if (++i == a.count) {
                i = 0;
                ++tile;
            }
        }
        if (tile != have_tile) g = group_of(a, plan, tile);
        const int id = g - 1, tokens = plan.tokens(g, tile);
        if (id < 0 && a.base[i] == a.y[i]) continue;
        const int R = a.R[i], M = a.M[i], col0 = c * kCols + warp * 32;
        const bool fresh = tile != have_tile || i != have_i;       // another tile or projection: its h
        if (fresh) {
            if (tile != have_tile) list_tile(a, plan, g, tile);
            have_tile = tile;
            have_i = i;
            rank = id < 0 ? 0 : rank_of(a, i, id);
        }
        // the next task's rows of B and base, into L2: a line of 128 bytes per lane and row
        if (col0 + kCols < M) {
            if (rank) prefetch_l2(a.b[i] + ((size_t)id * M + min(M - 1, col0 + kCols + lane)) * R);
            if (a.base[i])
                for (int t = lane; t < tokens; t += 32) prefetch_l2(a.base[i] + (size_t)plan.s_list[t] * M + col0 + kCols);
        }
        // B of the warp's columns, ranks r0 .. r0 + 63
        const bool odd = rank & 7;                   // a rank that ends inside a lane's 16 bytes
        auto load_b = [&](int r0, uint4 (&w)[2][4]) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int m = col0 + column(n, row), r = r0 + s * 32 + quad * 8;
                    w[s][n] = m < M && r < rank ? __ldg(reinterpret_cast<const uint4 *>(a.b[i] + ((size_t)id * M + m) * R + r))
                                                : make_uint4(0, 0, 0, 0);
                    if (odd && r + 8 > rank) w[s][n] = first_values(w[s][n], rank - r);
                }
        };
        auto load_base = [&](int m16, float4 (&v)[2][2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int tok = m16 * 16 + row + 8 * h;
                const float *src = a.base[i] && tok < tokens ? a.base[i] + (size_t)plan.s_list[tok] * M : nullptr;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = col0 + n * 16 + quad * 4;
                    v[n][h] = src && col < M ? *reinterpret_cast<const float4 *>(src + col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
        };
        uint4 w[2][4];
        load_b(0, w);
        float4 base[2][2];
        load_base(0, base);
        if (fresh) {
            __syncthreads();
            const int pad = (rank + 31) & ~31;
            const float scale = id < 0 ? 0.0f : (a.scale[i] ? __ldg(a.scale[i] + id) : 1.0f);
            const int rows16 = (tokens + 15) & ~15;
            for (int e = threadIdx.x; e < rows16 * (pad / 2); e += kW * 32) {
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
        }
        for (int m16 = 0; m16 * 16 < tokens; ++m16) {
            float4 now[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                now[n][0] = base[n][0];
                now[n][1] = base[n][1];
            }
            if ((m16 + 1) * 16 < tokens) load_base(m16 + 1, base);
            float acc[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
            for (int r0 = 0; r0 < rank; r0 += 64) {
                if (rank > 64) load_b(r0, w);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (r0 + s * 32 >= rank) break;
#pragma unroll
                    for (int z = 0; z < 3; ++z) {
                        const uint16_t *hp = s_h + z * plane + (m16 * 16 + row) * pitch + r0 + s * 32 + quad * 8;
                        const uint4 lo = *reinterpret_cast<const uint4 *>(hp), hi = *reinterpret_cast<const uint4 *>(hp + 8 * pitch);
                        const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma_bf16(acc[n], f0, w[s][n].x, w[s][n].y);
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma_bf16(acc[n], f1, w[s][n].z, w[s][n].w);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int tok = m16 * 16 + row + 8 * h;
                if (tok >= tokens) continue;
                float *dst = a.y[i] + (size_t)plan.s_list[tok] * M;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = col0 + n * 16 + quad * 4;
                    const float4 v = now[n][h];
                    if (col < M)
                        *reinterpret_cast<float4 *>(dst + col) =
                            make_float4(v.x + acc[2 * n][2 * h], v.y + acc[2 * n][2 * h + 1], v.z + acc[2 * n + 1][2 * h], v.w + acc[2 * n + 1][2 * h + 1]);
                }
            }
        }
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
    long long cols = 0;
    for (int i = 0; i < count; ++i) {
        most = std::max(most, a.R[i]);
        cols += (a.M[i] + kCols - 1) / kCols;
    }
    const int pitch = ((most + 31) & ~31) + 8;
    const size_t plan = Plan::bytes(a.adapters, piece);
    const size_t shrink_smem = (size_t)kW * kStages * kStageBytes + plan;
    const size_t expand_smem = (size_t)3 * kTok * pitch * 2 + plan;
    static bool set = false;
    if (!set) {
        TQ_CHECK(cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
        TQ_CHECK(cudaFuncSetAttribute(lora_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
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
        const int expand = (int)std::min<long long>(tiles * cols, 2 * sms);
        launch_pdl(lora_shrink_kernel, dim3(shrink), dim3(kW * 32), shrink_smem, a);
        launch_pdl(lora_expand_kernel, dim3(expand), dim3(kW * 32), expand_smem, a, pitch);
    }
    TQ_LAUNCH_CHECK("lora_expand_kernel");
    return 0;
}
