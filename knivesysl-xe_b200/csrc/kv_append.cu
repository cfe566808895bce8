// kv_append.cu — the new tokens' keys and values into a paged cache (x_kv_append).
//
// q, k and v arrive as the projections left them (fp32 rows). For every q and k head row h of a
// token at position p:
//   norm      h <- h * rsqrt(mean(h^2) + eps) * (1 + w)                      (optional, per head)
//   rotation  (a, b) <- (a cos - b sin, b cos + a sin), angle p * inv_freq[j],
//             pairs (j, j + rot/2), or (2j, 2j + 1) when interleaved; dims from rot on stay
// q goes out as bf16 rows, k and v to slot p of the request's pages as bf16 or e4m3 / scale. The
// angle is a product in 64 bits, reduced to half a turn there: at position 10^6 an fp32 product
// would be off by 0.06 rad. The only roundings to fewer bits than 32 are the stores.
//
// Nothing is read twice, so bytes bound it, and launch latency below some hundred tokens. A warp
// takes head rows of ONE token, so that its lanes' angles, page and slot serve all of them; a lane
// holds dim / 32 neighbouring values, which makes every load and store of a row one contiguous
// access of the warp, and a rotation partner sits in the same register of another lane (half
// split) or in the neighbouring register (interleaved).
#include "kv.cuh"

#include <algorithm>
#include <cudaTypedefs.h>

namespace tq {

namespace {

constexpr int kWarps = 8;
constexpr int kBatch = 4;             // head rows of a warp whose loads are under way together

struct AppendArgs {
    KvArgs kv;
    const float *q, *k, *v;
    size_t ldq, ldk, ldv;
    uint16_t *q_out;
    int q_heads;
    const float *inv_freq;
    int rot, interleaved;
    const uint16_t *q_norm, *k_norm;
    float eps;
    int parts, rows_per_warp;    // warps that share a token, head rows that each takes in turn
};

// The request of token t: the last r with start[r] <= t, 32 candidates per step.
__device__ __forceinline__ int find_request(const KvArgs &a, int t, int lane) {
    int lo = 0, n = a.count;                       // start[lo] <= t < start[lo + n] if anywhere
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int at = lo + lane * step;
        const bool below = lane * step < n && __ldg(a.start + at) <= t;
        const unsigned votes = __ballot_sync(0xffffffffu, below);
        const int last = votes ? 31 - __clz(votes) : 0;
        const int end = lo + n;
        lo += last * step;
        n = min(step, end - lo);
    }
    return lo;
}

template <int E>
__device__ __forceinline__ void load_row(const float *p, float (&x)[E]) {
    if constexpr (E == 2) {
        const float2 v = __ldg(reinterpret_cast<const float2 *>(p));
        x[0] = v.x; x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(p + i));
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
    }
}
template <int E>
__device__ __forceinline__ void store_bf16(uint16_t *p, const float (&x)[E]) {
    if constexpr (E == 2) *reinterpret_cast<uint32_t *>(p) = pack_bf16(x[0], x[1]);
    if constexpr (E == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    if constexpr (E == 8)
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                                   pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
template <int E>
__device__ __forceinline__ void store_e4m3(uint8_t *p, const float (&x)[E], float scale) {
    uint16_t h[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) h[i] = pack_e4m3(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale));
    if constexpr (E == 2) *reinterpret_cast<uint16_t *>(p) = h[0];
    if constexpr (E == 4) *reinterpret_cast<uint32_t *>(p) = h[0] | (uint32_t)h[1] << 16;
    if constexpr (E == 8)
        *reinterpret_cast<uint2 *>(p) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kWarps * 32) kv_append_kernel(const AppendArgs a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const unsigned number = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = (int)(number / (unsigned)a.parts);
    const int rows = a.q_heads + 2 * a.kv.heads;
    const int row0 = (int)(number % (unsigned)a.parts) * a.rows_per_warp;
    const int row1 = min(rows, row0 + a.rows_per_warp);
    pdl_wait();
    pdl_trigger();
    if (t >= a.kv.tokens || row0 >= rows) return;
    // the first rows' loads need only the token's number: they are under way while its request is looked up
    const int e0 = lane * E;
    auto source = [&](int row) -> const float * {
        if (row < a.q_heads) return a.q + (size_t)t * a.ldq + (size_t)row * D + e0;
        row -= a.q_heads;
        if (row < a.kv.heads) return a.k + (size_t)t * a.ldk + (size_t)row * D + e0;
        return a.v + (size_t)t * a.ldv + (size_t)(row - a.kv.heads) * D + e0;
    };
    float next[kBatch][E];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (first + i < row1) load_row<E>(source(first + i), next[i]);
    };
    load(row0);
    const int r = find_request(a.kv, t, lane);
    const KvRequest req = kv_request(a.kv, r);
    const int i = t - req.t0;
    if (i < 0 || i >= req.n) return;               // a row behind the last request
    const int pos = req.total - req.n + i;

    // this lane's cosines and sines, with the sign that the partner's product takes
    float cs[E], sn[E];
    const int half = a.rot >> 1;
    const bool turns = e0 < a.rot;                 // rot is a multiple of 16: whole lanes turn or not
#pragma unroll
    for (int e = 0; e < E; ++e) {
        cs[e] = 1.0f;
        sn[e] = 0.0f;
        if (turns && (!a.interleaved || !(e & 1))) {
            const int j = a.interleaved ? (e0 + e) >> 1 : (e0 + e < half ? e0 + e : e0 + e - half);
            // angle / pi in 64 bits, reduced to [-1, 1]
            double h = (double)pos * (double)__ldg(a.inv_freq + j) * 0.31830988618379067154;
            h -= 2.0 * rint(0.5 * h);
            sincospif((float)h, &sn[e], &cs[e]);
            if (!a.interleaved && e0 < half) sn[e] = -sn[e];
        }
    }
    // 1 + w of this lane's values
    float gq[E], gk[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        gq[e] = a.q_norm && row0 < a.q_heads ? 1.0f + __uint_as_float((uint32_t)__ldg(a.q_norm + e0 + e) << 16) : 1.0f;
        gk[e] = a.k_norm && row1 > a.q_heads ? 1.0f + __uint_as_float((uint32_t)__ldg(a.k_norm + e0 + e) << 16) : 1.0f;
    }
    const int partner = a.interleaved || !turns ? lane : (e0 < half ? lane + half / E : lane - half / E);

    // the cache slot, for the lanes' k and v rows (the head moves it by whole pages' rows)
    const long long slot = row1 > a.q_heads ? kv_row(a.kv, r, 0, pos) : -1;

    for (int first = row0; first < row1; first += kBatch) {
        float rowv[kBatch][E];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) rowv[i][e] = next[i][e];
        if (first + kBatch < row1) load(first + kBatch);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int row = first + b;
            if (row >= row1) break;
            float (&x)[E] = rowv[b];
            const bool is_q = row < a.q_heads, is_v = row >= a.q_heads + a.kv.heads;
            if (!is_v) {
                if (is_q ? a.q_norm : a.k_norm) {
                    float ss = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                    for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                    const float f = __frsqrt_rn(ss * (1.0f / D) + a.eps);
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = x[e] * f * (is_q ? gq[e] : gk[e]);
                }
                if (a.interleaved) {
                    if (turns)
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float u = x[e], v = x[e + 1];
                            x[e] = fmaf(u, cs[e], -(v * sn[e]));
                            x[e + 1] = fmaf(v, cs[e], u * sn[e]);
                        }
                } else if (a.rot) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float o = __shfl_sync(0xffffffffu, x[e], partner);
                        if (turns) x[e] = fmaf(x[e], cs[e], o * sn[e]);
                    }
                }
            }
            if (is_q) {
                if (a.q_out) store_bf16<E>(a.q_out + ((size_t)t * a.q_heads + row) * D + e0, x);
                continue;
            }
            if (slot < 0) continue;
            const int g = row - a.q_heads - (is_v ? a.kv.heads : 0);
            const size_t at = ((size_t)slot + (size_t)g * a.kv.page_size) * D + e0;
            uint8_t *pool = is_v ? a.kv.v : a.kv.k;
            if constexpr (E4M3) store_e4m3<E>(pool + at, x, is_v ? a.kv.v_scale : a.kv.k_scale);
            else store_bf16<E>(reinterpret_cast<uint16_t *>(pool) + at, x);
        }
    }
}

template <int D>
void launch(const AppendArgs &a, bool e4m3, dim3 grid) {
    if (e4m3) launch_pdl(kv_append_kernel<D, true>, grid, dim3(kWarps * 32), 0, a);
    else launch_pdl(kv_append_kernel<D, false>, grid, dim3(kWarps * 32), 0, a);
    TQ_LAUNCH_CHECK("kv_append_kernel");
}

}  // namespace

bool stream_is_capturing() {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(stream(), &st) != cudaSuccess || st != cudaStreamCaptureStatusNone;
}

int gpu_sms() {
    static int n = 0;
    if (!n) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, tq_device());
    return n > 0 ? n : 148;
}

bool tensor_map_2d(CUtensorMap &map, const void *data, int cols, long long rows, int box_rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    if (!encode || rows >= 0x7fffffffll) return false;      // rows are counted in 32 bits
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(data), dims, strides, boxes, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int kv_args(const tq_kv_cache_t *c, const tq_kv_batch_t *b, KvArgs &a) {
    if (!c || !b || !c->d_k || !c->d_v || c->pages <= 0 || c->page_size <= 0 || c->heads <= 0) return -1;
    if (c->e4m3 != 0 && c->e4m3 != 1) return -1;
    if (c->e4m3 && !(c->k_scale > 0.0f && c->v_scale > 0.0f && c->k_scale < INFINITY && c->v_scale < INFINITY)) return -1;
    if (b->count < 0 || b->tokens < 0 || b->max_new < 0 || b->max_pages < 0) return -2;
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return -3;
    // positions and page rows are counted in 32 bits, places in the pool in 64
    if ((long long)b->max_pages * c->page_size > 0x7fffff00ll) return -3;
    if (!aligned16(c->d_k) || !aligned16(c->d_v)) return -4;
    if (b->count && b->tokens && b->max_new && (!b->d_start || !b->d_kv_len || !b->d_pages || !b->max_pages)) return -2;
    a.k = static_cast<uint8_t *>(c->d_k);
    a.v = static_cast<uint8_t *>(c->d_v);
    a.pages = c->pages;
    a.page_size = c->page_size;
    a.heads = c->heads;
    a.dim = c->dim;
    a.k_scale = c->e4m3 ? c->k_scale : 1.0f;
    a.v_scale = c->e4m3 ? c->v_scale : 1.0f;
    a.start = b->d_start;
    a.kv_len = b->d_kv_len;
    a.page = b->d_pages;
    a.count = b->count;
    a.tokens = b->tokens;
    a.max_new = b->max_new;
    a.max_pages = b->max_pages;
    a.status = nullptr;
    return 0;
}

}  // namespace tq

int x_kv_append(const tq_kv_cache_t *cache, const tq_kv_batch_t *batch, const tq_rope_t *rope, const float *d_q,
                size_t ldq, int q_heads, uint16_t *d_q_out, const float *d_k, size_t ldk, const float *d_v,
                size_t ldv) {
    using namespace tq;
    AppendArgs a{};
    if (const int rc = kv_args(cache, batch, a.kv)) return rc;
    const int D = a.kv.dim;
    if (rope) {
        if (rope->rot_dim < 0 || rope->rot_dim > D || rope->rot_dim % 16) return -3;
        if (rope->rot_dim && !rope->d_inv_freq) return -1;
        if ((rope->d_q_norm || rope->d_k_norm) && !(rope->eps >= 0.0f)) return -1;
        a.inv_freq = rope->d_inv_freq;
        a.rot = rope->rot_dim;
        a.interleaved = rope->interleaved != 0;
        a.q_norm = rope->d_q_norm;
        a.k_norm = rope->d_k_norm;
        a.eps = rope->eps;
    }
    if (q_heads < 0 || (q_heads > 0) != (d_q != nullptr) || (q_heads > 0) != (d_q_out != nullptr)) return -2;
    if (q_heads > 65535 || a.kv.heads > 65535) return -3;
    if (!a.kv.count || !a.kv.tokens || !a.kv.max_new) return 0;
    if (!d_k || !d_v) return -2;
    if ((q_heads && ldq < (size_t)q_heads * D) || ldk < (size_t)a.kv.heads * D || ldv < (size_t)a.kv.heads * D) return -2;
    if ((q_heads && (!aligned16(d_q) || !aligned16(d_q_out) || ldq % 4)) || !aligned16(d_k) || !aligned16(d_v) || ldk % 4 ||
        ldv % 4)
        return -4;
    // the queries' rows are stored while other rows are being read
    const auto span = [&](size_t ld, int heads) { return ((a.kv.tokens - 1) * ld + (size_t)heads * D) * sizeof(float); };
    const size_t out_bytes = (size_t)a.kv.tokens * q_heads * D * sizeof(uint16_t);
    if (overlap(d_q_out, out_bytes, d_q, span(ldq, q_heads)) || overlap(d_q_out, out_bytes, d_k, span(ldk, a.kv.heads)) ||
        overlap(d_q_out, out_bytes, d_v, span(ldv, a.kv.heads)))
        return -2;
    if (!device_status_ready()) return -40;
    a.kv.status = device_status_word();
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.q_out = d_q_out;
    a.q_heads = q_heads;
    const int rows = q_heads + 2 * a.kv.heads;
    // As few warps a token as fill the GPU (32 an SM): the request, its page and the angles are looked up once a warp,
    // which costs as much as some ten head rows. 2156 tokens of 56 rows: 28 us with 8 warps a token.
    const long long want = 32ll * gpu_sms();
    a.parts = (int)std::min<long long>(rows, (want + a.kv.tokens - 1) / a.kv.tokens);
    a.rows_per_warp = (rows + a.parts - 1) / a.parts;
    const long long warps = (long long)a.kv.tokens * a.parts;
    if (warps > 0x7fffffffll) return -3;
    const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps));
    if (D == 64) launch<64>(a, cache->e4m3 != 0, grid);
    else if (D == 128) launch<128>(a, cache->e4m3 != 0, grid);
    else launch<256>(a, cache->e4m3 != 0, grid);
    return 0;
}
