// q4_cache.cu -- entry points of the 4-bit KV cache (format: q4.cuh) and its small
// kernels: import and export of rows, accumulated weights, and the rotary positions
// of three axes as a pass of their own.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>

#include "q4.cuh"

namespace dz {

void rope_axes_set(RopeAxes& a, const int32_t sections[3], bool interleaved, double base) {
    for (int i = 0; i < ROPE / 2; ++i) {
        int axis;
        if (interleaved)   // t h w t h w ..., time where height or width has used up its pairs
            axis = i % 3 == 1 && i < 3 * sections[1] ? 1 : (i % 3 == 2 && i < 3 * sections[2] ? 2 : 0);
        else
            axis = i < sections[0] ? 0 : (i < sections[0] + sections[1] ? 1 : 2);
        a.axis[i] = (uint8_t)axis;
        a.turn[i] = std::pow(base, -2.0 * i / ROPE) / 3.14159265358979323846;
    }
}

// The power of two that brings the largest q that these norm weights allow, 16 |w| sqrt(2) / 16 log2 e = 2.05 |w| for a row
// of one value and its rotation, to 2^14 .. 2^15: f16 then holds every query, small weights' too.
float query_scale(const float* q_norm) {
    float top = 0.0f;
    for (int i = 0; i < HD; ++i)
        if (std::isfinite(q_norm[i])) top = std::max(top, std::fabs(q_norm[i]));
    int e = 0;
    std::frexp(2.05 * top, &e);
    return top > 0.0f ? std::ldexp(1.0f, std::min(std::max(15 - e, -120), 120)) : 1.0f;
}

// An allocation is no work of the stream: it may be made while a graph is captured, on this thread or another
// (the buffer stays until the caches go, so the graph may hold it).
static cudaError_t alloc_uncaptured(void** p, size_t bytes) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    e = cudaMalloc(p, bytes);
    const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaErrorMemoryAllocation) cudaGetLastError();
    return e != cudaSuccess ? e : back;
}

cudaError_t ensure_q4_scratch(dz_ctx* ctx, size_t bytes) {
    if (ctx->q4_scratch_bytes >= bytes) return cudaSuccess;
    try {
        ctx->q4_retired.reserve(ctx->q4_retired.size() + 1);
    } catch (const std::exception&) {
        return cudaErrorMemoryAllocation;
    }
    // at least twice the size before, so that all the old ones together are smaller than the new one
    size_t size = std::max(bytes, 2 * ctx->q4_scratch_bytes);
    void* p = nullptr;
    cudaError_t e = alloc_uncaptured(&p, size);
    if (e == cudaErrorMemoryAllocation && size > bytes) e = alloc_uncaptured(&p, size = bytes);
    if (e != cudaSuccess) return e;
    if (ctx->q4_scratch) ctx->q4_retired.push_back(ctx->q4_scratch);
    ctx->q4_scratch = p;
    ctx->q4_scratch_bytes = size;
    return cudaSuccess;
}

namespace q4 {

// ---- rows as f32 ---------------------------------------------------------------------
// A list of row ranges, one per sequence: rows [first, first + count) of sequence sid go
// to output rows [row0, row0 + count).
struct Ranges {
    int B;
    int32_t sid[MAXB], first[MAXB];
    int32_t row0[MAXB + 1];
};
__device__ __forceinline__ int range_of(const int32_t* start, int B, int at) {   // last b with start[b] <= at
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= at) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// One warp per (row, kv head); a lane writes 4 dims of either half of K and V, whole lines a warp.
// 8192 rows (76 MB): 12.5 us, 6.1 TB/s.  With 8 dims a lane a store fills half sectors: 19 us;
// several heads to a warp, their loads ahead: 26 to 33 us.
__global__ void __launch_bounds__(256) q4_rows_kernel(Ranges d, int kvc, const Q4Slot* __restrict__ slots,
                                                      float* __restrict__ k, float* __restrict__ v) {
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (task >= (int64_t)d.row0[d.B] * kvc) return;
    const int row = (int)(task / kvc), kvh = (int)(task - (int64_t)row * kvc);
    const int b = range_of(d.row0, d.B, row);
    const int pos = d.first[b] + (row - d.row0[b]);
    const uint8_t* tile = slots[d.sid[b]].tile(kvh, pos >> 4);
    const size_t at = (size_t)task * HD + 4 * lane;
    uint32_t h[4][2];                            // K's halves, V's halves
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        get_k4(tile, pos & 15, lane, half, h[half]);
        get_v4(tile, pos & 15, lane, half, h[2 + half]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[i][0]));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h[i][1]));
        *reinterpret_cast<float4*>((i < 2 ? k : v) + at + 128 * (i & 1)) = make_float4(x.x, x.y, y.x, y.y);
    }
}

// One block per (tile, kv head), a warp per position: rows [row0, len) from f32
// [row][kvc][256], the tile's other positions as they are.  k and v start at row `row0`
// (a multiple of 16).  The call is bound by the copies of its rows into the scratch.
__global__ void __launch_bounds__(512) q4_import_kernel(Q4Slot slot, int kvc, int64_t row0, int64_t len,
                                                        const float* __restrict__ k, const float* __restrict__ v) {
    __shared__ TileMerge merge;
    const int64_t t = blockIdx.x / kvc;
    const int kvh = (int)(blockIdx.x - t * kvc), p = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* tile = slot.tile(kvh, (row0 >> 4) + t);
    merge.begin();
    __syncthreads();
    const int64_t row = t * Q4_TILE + p;
    if (row0 + row < len) {
        const size_t at = ((size_t)row * kvc + kvh) * HD + 8 * lane;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = k[at + e];
            y[e] = v[at + e];
        }
        uint32_t code[8];
        uint32_t sb = quantise(x, code);
        put_k(tile, p, lane, code, sb);
        sb = quantise(y, code);
        merge.add(p, lane, code);
        put_v_scale(tile, p, lane, sb);
    }
    merge.end(tile, 0, (int)min((int64_t)Q4_TILE, len - row0 - t * Q4_TILE));
}

// ---- accumulated weights ---------------------------------------------------------------
// flat: sequence b's [kvc][len] behind those before it.  Grid (ceil(longest / 1024), kvc, B).
struct Weights {
    int32_t sid[MAXB], len[MAXB];
    int64_t at[MAXB];
};
__global__ void __launch_bounds__(256) q4_weights_copy_kernel(Weights d, int kvc, const Q4Slot* __restrict__ slots,
                                                              float* __restrict__ out, const float* __restrict__ in) {
    const int b = blockIdx.z, kvh = blockIdx.y, n = d.len[b];
    const Q4Slot slot = slots[d.sid[b]];
    float* w = slot.wts + (size_t)kvh * slot.cap;
    const size_t at = (size_t)d.at[b] + (size_t)kvh * n;
    for (int j = blockIdx.x * 1024 + threadIdx.x; j < min(n, (int)(blockIdx.x + 1) * 1024); j += 256) {
        if (in) w[j] = in[at + j];
        else out[at + j] = w[j];
    }
}
__global__ void __launch_bounds__(256) q4_weights_clear_kernel(Q4Slot slot, int kvc, int64_t len) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < len * kvc) slot.wts[(i / len) * slot.cap + i % len] = 0.0f;
}

// ---- rotary positions of three axes ------------------------------------------------------
// QK-RMSNorm, rotation and q's 1/16 for T tokens.  HBM bound: q's halves of q_gate and k
// read once, q and k written once.  The angle is reduced in f64, sine and cosine taken
// in f32.  k_out may be k: a row is loaded whole by the warp that writes it.
__device__ __forceinline__ void store_split(float* row, int lane, const float (&x)[8]) {
    *reinterpret_cast<float4*>(row + split_dim(lane, 0)) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(row + split_dim(lane, 1)) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store_split(__nv_bfloat16* row, int lane, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint2*>(row + split_dim(lane, 0)) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(row + split_dim(lane, 1)) = make_uint2(w[2], w[3]);
}

// A warp per token and share of its heads: grid (ceil(T / 8), shares).  Several rows are
// in flight per warp: reading one at a time held the pass at 4.3 TB/s.  32768 bf16 tokens
// (0.94 GB): 160.4 us, 5.9 TB/s, 0.89 of a plain copy's rate (7 rows: 164 us, 14: 221); 12000 f32 (0.69 GB): 112 us, 6.1.
constexpr int MROPE_ROWS = 4;
template <typename T>
__global__ void __launch_bounds__(256) qk_mrope_kernel(const __grid_constant__ RopeAxes axes, int kvc, int64_t n_tokens,
                                                       const int32_t* __restrict__ pos, const T* __restrict__ q_gate,
                                                       const T* k, const float* __restrict__ q_norm,
                                                       const float* __restrict__ k_norm, T* __restrict__ q_out, T* k_out,
                                                       float eps) {
    const int lane = threadIdx.x & 31, nq = GRP * kvc;
    const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= n_tokens) return;
    float2 cs[4];
    spread_pairs(rope_cs_f32(axes, lane, pos[3 * t], pos[3 * t + 1], pos[3 * t + 2]), cs, lane);
    float wq[8], wk[8];
    load_split(q_norm, lane, wq);
    load_split(k_norm, lane, wk);
#pragma unroll
    for (int e = 0; e < 8; ++e) wq[e] *= 0.0625f;
    static_assert(HQ + HKV <= 32, "a bit per head");
    const int heads = nq + kvc, share = (heads + gridDim.y - 1) / gridDim.y;
    const int h1 = min(heads, ((int)blockIdx.y + 1) * share);
    uint32_t far = 0;                            // heads whose row is out of range
    for (int h0 = blockIdx.y * share; h0 < h1; h0 += MROPE_ROWS) {
        SplitRow<T> in[MROPE_ROWS];
#pragma unroll
        for (int i = 0; i < MROPE_ROWS; ++i) {
            const int h = h0 + i;
            if (h < h1) in[i].load(h < nq ? q_gate + (t * nq + h) * QG_ROW : k + (t * kvc + (h - nq)) * HD, lane);
        }
#pragma unroll
        for (int i = 0; i < MROPE_ROWS; ++i) {
            const int h = h0 + i;
            if (h >= h1) break;
            float x[8];
            in[i].values(x);
            const bool near = h < nq ? norm_rotate_split(x, wq, cs, eps, lane) : norm_rotate_split(x, wk, cs, eps, lane);
            if (near) store_split(h < nq ? q_out + (t * nq + h) * HD : k_out + (t * kvc + (h - nq)) * HD, lane, x);
            else far |= 1u << h;
        }
    }
    for (; far; far &= far - 1) {
        const int h = __ffs(far) - 1;
        float x[8];
        load_split(h < nq ? q_gate + (t * nq + h) * QG_ROW : k + (t * kvc + (h - nq)) * HD, lane, x);
        if (h < nq) norm_rotate_far(x, wq, cs, eps, lane);
        else norm_rotate_far(x, wk, cs, eps, lane);
        store_split(h < nq ? q_out + (t * nq + h) * HD : k_out + (t * kvc + (h - nq)) * HD, lane, x);
    }
}

}  // namespace q4

// ---- host ------------------------------------------------------------------------------
namespace {

dz_status fail(dz_ctx* ctx, dz_status st, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    ctx->err = buf;
    return st;
}
dz_status cuda_fail(dz_ctx* ctx, cudaError_t e, const char* what) {
    cudaGetLastError();   // reported here: the next call's launch check must not find it again
    return fail(ctx, e == cudaErrorMemoryAllocation ? DZ_ENOMEM : DZ_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}
#define Q4_CUDA(call)                                            \
    do {                                                         \
        const cudaError_t e_ = (call);                           \
        if (e_ != cudaSuccess) return cuda_fail(ctx, e_, #call); \
    } while (0)

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// no C++ exception leaves a C entry point: what can be thrown here is a failed or too large
// allocation of a host vector
template <typename F>
dz_status guarded(dz_ctx* ctx, F&& body) {
    if (!ctx) return DZ_EINVAL;
    try {
        return body();
    } catch (const std::exception&) {
        ctx->err.assign("out of memory");   // short enough to need none
        return DZ_ENOMEM;
    }
}

// layer, cache kind and sequence list of a call on 4-bit caches
dz_status check_layer(dz_ctx* ctx, int layer, bool params) {
    if (layer < 0 || layer >= (int)ctx->layers.size()) return fail(ctx, DZ_EINVAL, "bad layer %d", layer);
    const LayerState& L = ctx->layers[layer];
    if (!L.is_attn) return fail(ctx, DZ_EINVAL, "layer %d is not a full-attention layer", layer);
    if (params && !L.params_set) return fail(ctx, DZ_ESTATE, "layer %d has no parameters", layer);
    return DZ_OK;
}
dz_status check_seqs(dz_ctx* ctx, int B, const int32_t* ids, const char* what) {
    if (B <= 0 || !ids) return fail(ctx, DZ_EINVAL, "B must be positive and %s non-null", what);
    if (!ctx->q4) return fail(ctx, DZ_ESTATE, "no 4-bit cache: call dz_cache_create_q4 first");
    std::vector<char> seen(ctx->n_seqs, 0);
    for (int b = 0; b < B; ++b) {
        if (ids[b] < 0 || ids[b] >= ctx->n_seqs) return fail(ctx, DZ_EINVAL, "%s[%d]=%d out of range", what, b, ids[b]);
        if (seen[ids[b]]) return fail(ctx, DZ_EINVAL, "%s[%d]=%d repeated in one call", what, b, ids[b]);
        seen[ids[b]] = 1;
    }
    return DZ_OK;
}
dz_status check_tracked(dz_ctx* ctx) {
    if (!ctx->q4_track)
        return fail(ctx, DZ_ESTATE, "the caches accumulate no weights: dz_cache_create_q4 with track_weights");
    return DZ_OK;
}

}  // namespace

// Import and export are synchronous, as for f32 caches; host or device pointers.  The
// rows pass through device scratch 4096 at a time.
static constexpr int64_t IO_ROWS = 4096;

dz_status q4_import(dz_ctx* ctx, int layer, int seq, const float* k, const float* v, int64_t len) {
    LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count;
    const size_t row = (size_t)kvc * HD;
    Q4_CUDA(cudaDeviceSynchronize());
    if (len > 0) Q4_CUDA(ensure_q4_scratch(ctx, 2 * row * std::min(len, IO_ROWS) * sizeof(float)));
    float* dk = static_cast<float*>(ctx->q4_scratch);
    for (int64_t r0 = 0; r0 < len; r0 += IO_ROWS) {
        const int64_t n = std::min(IO_ROWS, len - r0);
        float* dv = dk + n * row;
        Q4_CUDA(cudaMemcpy(dk, k + r0 * row, n * row * sizeof(float), cudaMemcpyDefault));
        Q4_CUDA(cudaMemcpy(dv, v + r0 * row, n * row * sizeof(float), cudaMemcpyDefault));
        const int64_t blocks = (n + Q4_TILE - 1) / Q4_TILE * kvc;
        q4::q4_import_kernel<<<(unsigned)blocks, 512>>>(L.h_q4[seq], kvc, r0, r0 + n, dk, dv);
        Q4_CUDA(cudaGetLastError());
    }
    if (ctx->q4_track && len > 0) {
        q4::q4_weights_clear_kernel<<<(unsigned)((len * kvc + 255) / 256), 256>>>(L.h_q4[seq], kvc, len);
        Q4_CUDA(cudaGetLastError());
    }
    Q4_CUDA(cudaDeviceSynchronize());
    return DZ_OK;
}

dz_status q4_export(dz_ctx* ctx, int layer, int seq, float* k, float* v) {
    LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count;
    const int64_t len = L.len[seq];
    const size_t row = (size_t)kvc * HD;
    Q4_CUDA(cudaDeviceSynchronize());
    Q4_CUDA(ensure_q4_scratch(ctx, 2 * row * std::min(len, IO_ROWS) * sizeof(float)));
    float* dk = static_cast<float*>(ctx->q4_scratch);
    q4::Ranges d;
    d.B = 1;
    d.sid[0] = seq;
    for (int64_t r0 = 0; r0 < len; r0 += IO_ROWS) {
        const int64_t n = std::min(IO_ROWS, len - r0);
        float* dv = dk + n * row;
        d.first[0] = (int32_t)r0;
        d.row0[0] = 0;
        d.row0[1] = (int32_t)n;
        q4::q4_rows_kernel<<<(unsigned)((n * kvc + 7) / 8), 256>>>(d, kvc, L.d_q4, dk, dv);
        Q4_CUDA(cudaGetLastError());
        Q4_CUDA(cudaMemcpy(k + r0 * row, dk, n * row * sizeof(float), cudaMemcpyDefault));
        Q4_CUDA(cudaMemcpy(v + r0 * row, dv, n * row * sizeof(float), cudaMemcpyDefault));
    }
    Q4_CUDA(cudaDeviceSynchronize());
    return DZ_OK;
}

}  // namespace dz

using namespace dz;

extern "C" {

dz_status dz_set_rope_axes(dz_ctx* ctx, const int32_t* sections, int interleaved) {
    if (!ctx) return DZ_EINVAL;
    if (!sections) return fail(ctx, DZ_EINVAL, "null sections");
    int64_t sum = 0;
    for (int i = 0; i < 3; ++i) {
        if (sections[i] < 0) return fail(ctx, DZ_EINVAL, "sections[%d]=%d is negative", i, sections[i]);
        sum += sections[i];
    }
    if (sum != ROPE / 2) return fail(ctx, DZ_EINVAL, "the sections sum to %lld, not to %d pairs", (long long)sum, ROPE / 2);
    // every third pair from 1 (height) and from 2 (width): 11 and 10 of them below 32
    if (interleaved && (sections[1] > 11 || sections[2] > 10))
        return fail(ctx, DZ_EINVAL, "interleaved sections hold at most 11 pairs of height and 10 of width (%d, %d)",
                    sections[1], sections[2]);
    rope_axes_set(ctx->axes, sections, interleaved != 0, ctx->cfg.rope_freq_base);
    return DZ_OK;
}

}  // extern "C"

template <typename T>
static dz_status qk_mrope(dz_ctx* ctx, int layer, int64_t n, const int32_t* pos, const T* q_gate, const T* k, T* q_out,
                          T* k_out, void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, true);
        if (st != DZ_OK) return st;
        if (n < 1 || n > INT32_MAX) return fail(ctx, DZ_EINVAL, "T=%lld outside 1..2^31-1", (long long)n);
        if (!pos || !q_gate || !k || !q_out || !k_out) return fail(ctx, DZ_EINVAL, "null tensor");
        if (!aligned16(q_gate) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out))
            return fail(ctx, DZ_EINVAL, "q_gate, k, q_out and k_out must be 16-byte aligned");
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        const LayerState& L = ctx->layers[layer];
        const int kvc = ctx->cfg.kv_head_count;
        // Few tokens: a warp per head, so that their latencies overlap, while that leaves at most 20
        // warps per SM (f32, 64 tokens: 3.5 us, 4.8 with 4 shares; 200: 7.6 and 5.0); then 4 shares, up
        // to 40 (1200: 14.5 us, 16.5 with one; 2368: 29.6 and 24.8); then one share.
        const int heads = GRP * kvc + kvc;
        const int shares = n * heads <= 20 * ctx->n_sm ? heads : (n * 4 <= 40 * ctx->n_sm ? 4 : 1);
        q4::qk_mrope_kernel<T><<<dim3((unsigned)((n + 7) / 8), shares), 256, 0, static_cast<cudaStream_t>(stream)>>>(
            ctx->axes, kvc, n, pos, q_gate, k, L.q_norm, L.k_norm, q_out, k_out, ctx->cfg.rms_eps);
        Q4_CUDA(cudaGetLastError());
        ctx->last_launches = 1;
        return DZ_OK;
    });
}

extern "C" {

dz_status dz_qk_mrope(dz_ctx* ctx, int layer, int64_t T, const int32_t* pos, const float* q_gate, const float* k,
                      float* q_out, float* k_out, void* stream) {
    return qk_mrope(ctx, layer, T, pos, q_gate, k, q_out, k_out, stream);
}

dz_status dz_qk_mrope_bf16(dz_ctx* ctx, int layer, int64_t T, const int32_t* pos, const uint16_t* q_gate,
                           const uint16_t* k, uint16_t* q_out, uint16_t* k_out, void* stream) {
    using B = __nv_bfloat16;
    return qk_mrope(ctx, layer, T, pos, reinterpret_cast<const B*>(q_gate), reinterpret_cast<const B*>(k),
                    reinterpret_cast<B*>(q_out), reinterpret_cast<B*>(k_out), stream);
}

dz_status dz_gqa_decode_q4(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, const int32_t* pos,
                           const float* q_gate, const float* k, const float* v, float* out, void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, true);
        if (st != DZ_OK || (st = check_seqs(ctx, B, seq_ids, "seq_ids")) != DZ_OK) return st;
        LayerState& L = ctx->layers[layer];
        for (int b = 0; b < B; ++b)
            if (L.len[seq_ids[b]] + 1 > L.h_q4[seq_ids[b]].cap)
                return fail(ctx, DZ_ESTATE, "KV cache of seq %d is full (cap %lld)", seq_ids[b],
                            (long long)L.h_q4[seq_ids[b]].cap);
        for (int b = 0; pos && b < 3 * B; ++b)
            if (pos[b] < 0) return fail(ctx, DZ_EINVAL, "pos[%d][%d]=%d is negative", b / 3, b % 3, pos[b]);
        if (!q_gate || !k || !v || !out) return fail(ctx, DZ_EINVAL, "null tensor");
        if (!aligned16(q_gate) || !aligned16(k) || !aligned16(v))
            return fail(ctx, DZ_EINVAL, "q_gate, k and v must be 16-byte aligned");
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
        int launches = 0;
        for (int b0 = 0; b0 < B; b0 += MAXB) {
            Q4Rows d;
            Q4Pos p3;
            d.B = std::min(MAXB, B - b0);
            d.kvc = kvc;
            d.cum[0] = 0;
            for (int b = 0; b < d.B; ++b) {
                d.sid[b] = seq_ids[b0 + b];
                d.len[b] = (int32_t)L.len[d.sid[b]];
                for (int i = 0; i < 3; ++i) p3.p[b][i] = pos ? pos[3 * (b0 + b) + i] : d.len[b];
                d.cum[b + 1] = d.cum[b] + (int32_t)(((int64_t)d.len[b] + Q4_TILE) / Q4_TILE);
            }
            if (q4_decode_runs(ctx->n_sm) + d.B * kvc > ctx->part_items)   // cannot happen under decode_items_bound
                return fail(ctx, DZ_ESTATE, "the partials of %d sequences exceed the scratch (%lld)", d.B,
                            (long long)ctx->part_items);
            Q4_CUDA(launch_q4_decode(ctx, layer, d, p3, q_gate + (size_t)b0 * nq * QG_ROW, k + (size_t)b0 * kvc * HD,
                                     v + (size_t)b0 * kvc * HD, out + (size_t)b0 * nq * HD,
                                     static_cast<cudaStream_t>(stream), &launches));
        }
        for (int b = 0; b < B; ++b) L.len[seq_ids[b]] += 1;
        ctx->last_launches = launches;
        return DZ_OK;
    });
}

}  // extern "C"

template <typename T>
static dz_status gqa_prefill(dz_ctx* ctx, int layer, int n_seqs, const int32_t* seq_ids, const int64_t* T_new,
                             const int32_t* pos, const T* q_gate, const T* k, const T* v, T* out, void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, true);
        if (st != DZ_OK || (st = check_seqs(ctx, n_seqs, seq_ids, "seq_ids")) != DZ_OK) return st;
        if (!T_new) return fail(ctx, DZ_EINVAL, "null T");
        const LayerState& L = ctx->layers[layer];
        int64_t total = 0;
        for (int i = 0; i < n_seqs; ++i) {
            const int64_t len = L.len[seq_ids[i]], cap = L.h_q4[seq_ids[i]].cap;
            if (T_new[i] < 0) return fail(ctx, DZ_EINVAL, "T[%d]=%lld is negative", i, (long long)T_new[i]);
            if (T_new[i] > cap - len)
                return fail(ctx, DZ_ESTATE, "prefill of %lld tokens overflows the KV cache of seq %d (len %lld, cap %lld)",
                            (long long)T_new[i], seq_ids[i], (long long)len, (long long)cap);
            total += T_new[i];
        }
        if (total < 1 || total > INT32_MAX) return fail(ctx, DZ_EINVAL, "%lld tokens outside 1..2^31-1", (long long)total);
        if (!q_gate || !k || !v || !out) return fail(ctx, DZ_EINVAL, "null tensor");
        if (!aligned16(q_gate) || !aligned16(k) || !aligned16(v) || !aligned16(out))
            return fail(ctx, DZ_EINVAL, "q_gate, k, v and out must be 16-byte aligned");
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        int launches = 0;
        Q4_CUDA(launch_q4_prefill(ctx, layer, n_seqs, seq_ids, T_new, pos, q_gate, k, v, out,
                                  static_cast<cudaStream_t>(stream), &launches));
        ctx->last_launches = launches;
        return DZ_OK;
    });
}

extern "C" {

dz_status dz_gqa_prefill_q4(dz_ctx* ctx, int layer, int n_seqs, const int32_t* seq_ids, const int64_t* T,
                            const int32_t* pos, const float* q_gate, const float* k, const float* v, float* out,
                            void* stream) {
    return gqa_prefill(ctx, layer, n_seqs, seq_ids, T, pos, q_gate, k, v, out, stream);
}

dz_status dz_gqa_prefill_q4_bf16(dz_ctx* ctx, int layer, int n_seqs, const int32_t* seq_ids, const int64_t* T,
                                 const int32_t* pos, const uint16_t* q_gate, const uint16_t* k, const uint16_t* v,
                                 uint16_t* out, void* stream) {
    return gqa_prefill(ctx, layer, n_seqs, seq_ids, T, pos, q_gate, k, v, out, stream);
}

dz_status dz_kv_rows_q4(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, const int64_t* first,
                        const int64_t* count, float* k, float* v, void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, false);
        if (st != DZ_OK || (st = check_seqs(ctx, B, seq_ids, "seq_ids")) != DZ_OK) return st;
        if (!first || !count) return fail(ctx, DZ_EINVAL, "null argument");
        if (!aligned16(k) || !aligned16(v)) return fail(ctx, DZ_EINVAL, "k and v must be 16-byte aligned");
        const LayerState& L = ctx->layers[layer];
        int64_t total = 0;
        for (int b = 0; b < B; ++b) {
            const int64_t len = L.len[seq_ids[b]];
            if (first[b] < 0 || count[b] < 0 || first[b] > len || count[b] > len - first[b])
                return fail(ctx, DZ_EINVAL, "rows [%lld, +%lld) of seq %d outside its %lld", (long long)first[b],
                            (long long)count[b], seq_ids[b], (long long)len);
            total += count[b];
        }
        if (total > 0 && (!k || !v)) return fail(ctx, DZ_EINVAL, "null tensor");
        if (total > INT32_MAX) return fail(ctx, DZ_EINVAL, "%lld rows exceed 2^31-1 per call", (long long)total);
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        const int kvc = ctx->cfg.kv_head_count;
        int launches = 0;
        for (int b0 = 0; b0 < B; b0 += MAXB) {
            q4::Ranges d;
            d.B = std::min(MAXB, B - b0);
            d.row0[0] = 0;
            for (int b = 0; b < d.B; ++b) {
                d.sid[b] = seq_ids[b0 + b];
                d.first[b] = (int32_t)first[b0 + b];
                d.row0[b + 1] = d.row0[b] + (int32_t)count[b0 + b];
            }
            const int64_t rows = d.row0[d.B];
            if (rows > 0) {
                q4::q4_rows_kernel<<<(unsigned)((rows * kvc + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                    d, kvc, L.d_q4, k, v);
                Q4_CUDA(cudaGetLastError());
                ++launches;
            }
            k += (size_t)rows * kvc * HD;
            v += (size_t)rows * kvc * HD;
        }
        ctx->last_launches = launches;
        return DZ_OK;
    });
}

static dz_status weights_copy(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, float* out, const float* in,
                              void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, false);
        if (st != DZ_OK || (st = check_seqs(ctx, B, seq_ids, "seq_ids")) != DZ_OK ||
            (st = check_tracked(ctx)) != DZ_OK)
            return st;
        const LayerState& L = ctx->layers[layer];
        for (int b = 0; b < B; ++b)
            if (L.len[seq_ids[b]] > 0 && !out && !in) return fail(ctx, DZ_EINVAL, "null tensor");
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        const int kvc = ctx->cfg.kv_head_count;
        int launches = 0;
        int64_t at = 0;
        for (int b0 = 0; b0 < B; b0 += MAXB) {
            q4::Weights d;
            const int nb = std::min(MAXB, B - b0);
            int longest = 0;
            for (int b = 0; b < nb; ++b) {
                d.sid[b] = seq_ids[b0 + b];
                d.len[b] = (int32_t)L.len[d.sid[b]];
                d.at[b] = at;
                at += (int64_t)kvc * d.len[b];
                longest = std::max(longest, d.len[b]);
            }
            if (longest == 0) continue;
            q4::q4_weights_copy_kernel<<<dim3((longest + 1023) / 1024, kvc, nb), 256, 0,
                                         static_cast<cudaStream_t>(stream)>>>(d, kvc, L.d_q4, out, in);
            Q4_CUDA(cudaGetLastError());
            ++launches;
        }
        ctx->last_launches = launches;
        return DZ_OK;
    });
}

dz_status dz_kv_weights_q4(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, float* out, void* stream) {
    return weights_copy(ctx, layer, B, seq_ids, out, nullptr, stream);
}

dz_status dz_kv_set_weights_q4(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, const float* weights,
                               void* stream) {
    return weights_copy(ctx, layer, B, seq_ids, nullptr, weights, stream);
}

dz_status dz_kv_evict_q4(dz_ctx* ctx, int layer, int B, const int32_t* seq_ids, const int32_t* into,
                         const int64_t* keep, const int64_t* recent, int32_t* kept, void* stream) {
    return guarded(ctx, [&]() -> dz_status {
        dz_status st = check_layer(ctx, layer, false);
        if (st != DZ_OK || (st = check_seqs(ctx, B, seq_ids, "seq_ids")) != DZ_OK ||
            (into && (st = check_seqs(ctx, B, into, "into")) != DZ_OK) || (st = check_tracked(ctx)) != DZ_OK)
            return st;
        if (!keep || !recent) return fail(ctx, DZ_EINVAL, "null argument");
        LayerState& L = ctx->layers[layer];
        const int32_t* dst = into ? into : seq_ids;
        std::vector<int> source_of(ctx->n_seqs, -1);
        for (int b = 0; b < B; ++b) source_of[seq_ids[b]] = b;
        int64_t total = 0;
        for (int b = 0; b < B; ++b) {
            const int64_t n = L.len[seq_ids[b]], k = std::min(keep[b], n);
            if (keep[b] < 1 || recent[b] < 0 || recent[b] > keep[b])
                return fail(ctx, DZ_EINVAL, "keep[%d]=%lld, recent[%d]=%lld: need keep >= 1 and 0 <= recent <= keep", b,
                            (long long)keep[b], b, (long long)recent[b]);
            if (source_of[dst[b]] >= 0 && source_of[dst[b]] != b)
                return fail(ctx, DZ_EINVAL, "into[%d]=%d is a source of the same call", b, dst[b]);
            if (k > L.h_q4[dst[b]].cap)
                return fail(ctx, DZ_ESTATE, "%lld kept rows exceed the capacity %lld of seq %d", (long long)k,
                            (long long)L.h_q4[dst[b]].cap, dst[b]);
            total += k;
        }
        if (total * ctx->cfg.kv_head_count > INT32_MAX)
            return fail(ctx, DZ_EINVAL, "%lld kept rows exceed 2^31-1 indices per call", (long long)total);
        DeviceGuard g(ctx->device);
        if (!g.ok) return fail(ctx, DZ_ECUDA, "cudaSetDevice(%d) failed", ctx->device);
        int launches = 0;
        Q4_CUDA(launch_q4_evict(ctx, layer, B, seq_ids, dst, keep, recent, kept, static_cast<cudaStream_t>(stream),
                                &launches));
        std::vector<int64_t> n(B);
        for (int b = 0; b < B; ++b) n[b] = std::min(keep[b], L.len[seq_ids[b]]);
        for (int b = 0; b < B; ++b) {
            if (dst[b] == seq_ids[b] && n[b] == L.len[dst[b]]) continue;   // nothing moved
            L.len[dst[b]] = n[b];
            kv_lowered(ctx, layer, dst[b], 0);                             // rows rewritten from 0
        }
        ctx->last_launches = launches;
        return DZ_OK;
    });
}

}  // extern "C"
