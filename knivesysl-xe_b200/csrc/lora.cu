// lora.cu — low-rank adapters of many requests beside a shared projection (x_lora_add).
//
//   y[t] = base[t] + scale[a] (x[t] A[a]^T) B[a]^T,  a = adapter[t];  y[t] = base[t] without one
//
// in two launches for up to four projections that share x: "shrink" h = x A^T (rank values a token)
// and "expand" y = base + h B^T. Both work on tiles of up to 16 tokens of ONE adapter, whatever
// places the tokens have in the batch: a tile is the m16 side of an mma, its adapter's rows the n8
// side, so an adapter is read once per 16 of its tokens and never for the others. Each CTA sorts the
// batch's adapter numbers into tiles itself (they are few), so there is no launch for that.
//
// Bytes bound both: x and the adapters in shrink, base, y and the adapters in expand; 2 rank
// operations a value of x or y are far below that. x and h are fp32 and enter the bf16 tensor core
// as three bf16 terms, all 24 bits of them: exact up to the fp32 sums. The dimension that is summed is read in
// the order that suits the loads: a lane takes 16 bytes (8 neighbouring values) of a row, which are
// its share of two k16 steps, the same on both sides, so neither side passes through shared memory.
#include "kv.cuh"

#include <algorithm>

namespace tq {

namespace {

constexpr int kW = 8;                 // warps of a CTA
constexpr int kTok = 16;              // tokens of a tile
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
    int tiles_max;
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

// Adapter -1 counts as group 0, adapter id as group id + 1. s_off[g] = first tile of group g.
// Shared memory: (adapters + 2) + 1 ints, then kTok of the tile's tokens.
__device__ void plan(const LoraArgs &a, int *s_off) {
    const int groups = a.adapters + 1;
    for (int g = threadIdx.x; g <= groups; g += kW * 32) s_off[g] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < a.T; t += kW * 32) atomicAdd(s_off + adapter_of(a, t) + 1, 1);
    __syncthreads();
    if (threadIdx.x < 32) {                          // exclusive scan of the groups' tiles
        int base = 0;
        for (int g0 = 0; g0 <= groups; g0 += 32) {
            const int g = g0 + threadIdx.x;
            const int n = g < groups ? (s_off[g] + kTok - 1) / kTok : 0;
            int s = n;
            for (int off = 1; off < 32; off <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, s, off);
                if ((int)threadIdx.x >= off) s += o;
            }
            if (g <= groups) s_off[g] = base + s - n;
            base += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    __syncthreads();
}
// The group of tile x (s_off[0..groups] ascending).
__device__ __forceinline__ int group_of(const LoraArgs &a, const int *s_off, int x) {
    int lo = 0, hi = a.adapters + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_off[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Tokens of tile x into list[0..15] (one warp; -1 behind the last): the adapter's tokens number
// 16 i .. 16 i + 15 in ascending order.
__device__ void tile_tokens(const LoraArgs &a, int id, int skip, int *list, int lane) {
    if (lane < kTok) list[lane] = -1;
    __syncwarp();
    int seen = 0;
    for (int t0 = 0; t0 < a.T && seen < skip + kTok; t0 += 32) {
        const int t = t0 + lane;
        const bool hit = t < a.T && adapter_of(a, t) == id;
        const unsigned votes = __ballot_sync(0xffffffffu, hit);
        const int at = seen + __popc(votes & ((1u << lane) - 1)) - skip;
        if (hit && at >= 0 && at < kTok) list[at] = t;
        seen += __popc(votes);
    }
    __syncwarp();
}

// ---- shrink ------------------------------------------------------------------------------------
// A task is (tile, projection, part of K); the warps of a CTA take slices of the part and add their
// sums through shared memory. A lane's loads: 32 bytes of x for each of its two tokens and 16 bytes
// of A for each group of 8 ranks, per 32 values of K.
constexpr int kNB = 8;                // groups of 8 ranks per pass

__global__ void __launch_bounds__(kW * 32) lora_shrink_kernel(const LoraArgs a) {
    extern __shared__ int s_off[];
    __shared__ int s_list[kTok];
    __shared__ float s_sum[kW][kTok][kNB * 8 + 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    pdl_wait();
    pdl_trigger();
    plan(a, s_off);
    const int tile0 = s_off[1], tiles = s_off[a.adapters + 1] - tile0;      // group 0 has no product
    const int width = a.hoff[a.count];
    const int per = a.count * a.splits;
    for (int task = blockIdx.x; task < tiles * per; task += gridDim.x) {
        const int tile = tile0 + task / per, i = task % per / a.splits, part = task % a.splits;
        const int id = group_of(a, s_off, tile) - 1;
        if (warp == 0) tile_tokens(a, id, (tile - s_off[id + 1]) * kTok, s_list, lane);
        __syncthreads();
        const int rank = rank_of(a, i, id), R = a.R[i], K32 = a.K / 32;
        const int k0 = (int)((long long)K32 * part / a.splits), k1 = (int)((long long)K32 * (part + 1) / a.splits);
        const int w0 = k0 + (k1 - k0) * warp / kW, w1 = k0 + (k1 - k0) * (warp + 1) / kW;
        const int t_lo = s_list[row], t_hi = s_list[row + 8];
        const float *x_lo = a.x + (size_t)max(t_lo, 0) * a.K + quad * 8, *x_hi = a.x + (size_t)max(t_hi, 0) * a.K + quad * 8;
        for (int r0 = 0; r0 < rank; r0 += kNB * 8) {
            const int nb = min(kNB, (rank - r0 + 7) / 8);
            float acc[kNB][4];
#pragma unroll
            for (int n = 0; n < kNB; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
            const uint16_t *A = a.a[i] + ((size_t)id * R + r0 + row) * a.K + quad * 8;
            for (int k = w0; k < w1; ++k) {
                float4 xl[2] = {}, xh[2] = {};
                if (t_lo >= 0) {
                    xl[0] = __ldg(reinterpret_cast<const float4 *>(x_lo + k * 32));
                    xl[1] = __ldg(reinterpret_cast<const float4 *>(x_lo + k * 32 + 4));
                }
                if (t_hi >= 0) {
                    xh[0] = __ldg(reinterpret_cast<const float4 *>(x_hi + k * 32));
                    xh[1] = __ldg(reinterpret_cast<const float4 *>(x_hi + k * 32 + 4));
                }
                uint4 w[kNB];
#pragma unroll
                for (int n = 0; n < kNB; ++n)
                    w[n] = n < nb && r0 + n * 8 + row < rank
                               ? __ldg(reinterpret_cast<const uint4 *>(A + (size_t)n * 8 * a.K + k * 32))
                               : make_uint4(0, 0, 0, 0);
                uint32_t f[2][3][4];                  // [k16 step][term]
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    split3(xl[s].x, xl[s].y, f[s][0][0], f[s][1][0], f[s][2][0]);
                    split3(xh[s].x, xh[s].y, f[s][0][1], f[s][1][1], f[s][2][1]);
                    split3(xl[s].z, xl[s].w, f[s][0][2], f[s][1][2], f[s][2][2]);
                    split3(xh[s].z, xh[s].w, f[s][0][3], f[s][1][3], f[s][2][3]);
                }
#pragma unroll
                for (int n = 0; n < kNB; ++n)
                    if (n < nb) {
#pragma unroll
                        for (int z = 0; z < 3; ++z) {
                            mma_bf16(acc[n], f[0][z], w[n].x, w[n].y);
                            mma_bf16(acc[n], f[1][z], w[n].z, w[n].w);
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < kNB; ++n)
                if (n < nb) {
                    *reinterpret_cast<float2 *>(&s_sum[warp][row][n * 8 + quad * 2]) = make_float2(acc[n][0], acc[n][1]);
                    *reinterpret_cast<float2 *>(&s_sum[warp][row + 8][n * 8 + quad * 2]) = make_float2(acc[n][2], acc[n][3]);
                }
            __syncthreads();
            for (int e = threadIdx.x; e < kTok * nb * 8; e += kW * 32) {
                const int i_tok = e / (nb * 8), r = e % (nb * 8), t = s_list[i_tok];
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kW; ++w) s += s_sum[w][i_tok][r];
                if (t >= 0) a.h[((size_t)part * a.T + t) * width + a.hoff[i] + r0 + r] = s;
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

// The first n of 8 values, zeros behind them.
__device__ __forceinline__ uint4 first_values(uint4 v, int n) {
    auto word = [&](uint32_t x, int i) { return n >= 2 * i + 2 ? x : (n == 2 * i + 1 ? x & 0xffffu : 0u); };
    return make_uint4(word(v.x, 0), word(v.y, 1), word(v.z, 2), word(v.w, 3));
}

// ---- expand ------------------------------------------------------------------------------------
// A task is (tile, projection, 256 columns of y): 32 columns a warp. h of the tile, scaled and split
// into its three terms, lies in shared memory as [term][token][rank] for the whole CTA.
constexpr int kCols = 32 * kW;
constexpr int kHPitch = kMaxRank + 8;  // 16 bytes more than a multiple of 128: rows on different banks

__global__ void __launch_bounds__(kW * 32) lora_expand_kernel(const LoraArgs a) {
    extern __shared__ int s_off[];
    __shared__ int s_list[kTok];
    __shared__ __align__(16) uint16_t s_h[3][kTok][kHPitch];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, row = lane >> 2;
    pdl_wait();
    pdl_trigger();
    plan(a, s_off);
    const int tiles = s_off[a.adapters + 1], width = a.hoff[a.count];
    int blocks = 0;
    for (int i = 0; i < a.count; ++i) blocks += (a.M[i] + kCols - 1) / kCols;
    const long long total = (long long)tiles * blocks;
    const long long begin = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    int have_tile = -1, have_i = -1, rank = 0;
    for (long long task = begin; task < end; ++task) {
        const int tile = (int)(task / blocks);
        int c = (int)(task % blocks), i = 0;
        while (c >= (a.M[i] + kCols - 1) / kCols) c -= (a.M[i++] + kCols - 1) / kCols;
        const int id = group_of(a, s_off, tile) - 1;
        if (id < 0 && a.base[i] == a.y[i]) continue;
        if (tile != have_tile || i != have_i) {
            __syncthreads();
            if (tile != have_tile && warp == 0) tile_tokens(a, id, (tile - s_off[id + 1]) * kTok, s_list, lane);
            __syncthreads();
            have_tile = tile;
            have_i = i;
            rank = id < 0 ? 0 : rank_of(a, i, id);
            const int pad = (rank + 31) & ~31;
            const float scale = id < 0 ? 0.0f : (a.scale[i] ? __ldg(a.scale[i] + id) : 1.0f);
            for (int e = threadIdx.x; e < kTok * (pad / 2); e += kW * 32) {
                const int i_tok = e / (pad / 2), r = e % (pad / 2) * 2, t = s_list[i_tok];
                float v[2] = {0.0f, 0.0f};
                for (int x = 0; x < 2; ++x)
                    if (t >= 0 && r + x < rank) {
                        const float *h = a.h + (size_t)t * width + a.hoff[i] + r + x;
                        for (int s = 0; s < a.splits; ++s) v[x] += __ldcg(h + (size_t)s * a.T * width);
                        v[x] *= scale;
                    }
                uint32_t t0, t1, t2;
                split3(v[0], v[1], t0, t1, t2);
                *reinterpret_cast<uint32_t *>(&s_h[0][i_tok][r]) = t0;
                *reinterpret_cast<uint32_t *>(&s_h[1][i_tok][r]) = t1;
                *reinterpret_cast<uint32_t *>(&s_h[2][i_tok][r]) = t2;
            }
            __syncthreads();
        }
        const int R = a.R[i], M = a.M[i], col0 = c * kCols + warp * 32;
        const int t_lo = s_list[row], t_hi = s_list[row + 8];
        float acc[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int col = col0 + n * 8 + quad * 2;
            float2 lo = make_float2(0.0f, 0.0f), hi = lo;
            if (a.base[i] && col < M) {
                if (t_lo >= 0) lo = *reinterpret_cast<const float2 *>(a.base[i] + (size_t)t_lo * M + col);
                if (t_hi >= 0) hi = *reinterpret_cast<const float2 *>(a.base[i] + (size_t)t_hi * M + col);
            }
            acc[n][0] = lo.x; acc[n][1] = lo.y; acc[n][2] = hi.x; acc[n][3] = hi.y;
        }
        for (int r0 = 0; r0 < rank; r0 += 32) {
            uint4 w[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int m = col0 + n * 8 + row, r = r0 + quad * 8;
                w[n] = m < M && r < rank ? __ldg(reinterpret_cast<const uint4 *>(a.b[i] + ((size_t)id * M + m) * R + r))
                                         : make_uint4(0, 0, 0, 0);
                if (r + 8 > rank) w[n] = first_values(w[n], rank - r);
            }
#pragma unroll
            for (int z = 0; z < 3; ++z) {
                const uint4 lo = *reinterpret_cast<const uint4 *>(&s_h[z][row][r0 + quad * 8]);
                const uint4 hi = *reinterpret_cast<const uint4 *>(&s_h[z][row + 8][r0 + quad * 8]);
                const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    mma_bf16(acc[n], f0, w[n].x, w[n].y);
                    mma_bf16(acc[n], f1, w[n].z, w[n].w);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int col = col0 + n * 8 + quad * 2;
            if (col >= M) continue;
            if (t_lo >= 0) *reinterpret_cast<float2 *>(a.y[i] + (size_t)t_lo * M + col) = make_float2(acc[n][0], acc[n][1]);
            if (t_hi >= 0) *reinterpret_cast<float2 *>(a.y[i] + (size_t)t_hi * M + col) = make_float2(acc[n][2], acc[n][3]);
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
        if (w->K % 32 || w->M % 16 || w->rank % 8 || w->rank > kMaxRank || w->count > 2048) return -3;
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
    // at least one tile per 16 tokens, at most one per token or adapter more
    const int tiles = (T + kTok - 1) / kTok + std::min(T, a.adapters);
    a.tiles_max = tiles;
    const int k32 = a.K / 32;
    a.splits = std::max(1, std::min({16, 2 * sms / std::max(1, tiles * count), k32 / kW}));
    const size_t need = (size_t)a.splits * T * a.hoff[count];
    if (need > g_h_floats) {
        if (stream_is_capturing()) return -40;
        if (g_h) tq_dev_free(g_h);
        g_h = static_cast<float *>(tq_dev_alloc(need * sizeof(float), "lora.h"));
        g_h_floats = need;
    }
    a.h = g_h;
    a.status = device_status_word();
    const size_t smem = (size_t)(a.adapters + 2) * sizeof(int);
    const int shrink = (int)std::min<long long>((long long)tiles * count * a.splits, 2 * sms);
    long long cols = 0;
    for (int i = 0; i < count; ++i) cols += (a.M[i] + kCols - 1) / kCols;
    const int expand = (int)std::min<long long>(tiles * cols, 4 * sms);
    launch_pdl(lora_shrink_kernel, dim3(shrink), dim3(kW * 32), smem, a);
    launch_pdl(lora_expand_kernel, dim3(expand), dim3(kW * 32), smem, a);
    TQ_LAUNCH_CHECK("lora_expand_kernel");
    return 0;
}
