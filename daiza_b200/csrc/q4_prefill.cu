// q4_prefill.cu -- prompts into 4-bit KV caches: packed sequences of different lengths,
// rotary positions of three axes, causal attention over the held rows.
//
// Reference: Daiza-engine/src/model/forward.rs:599-721 (parallel GQA prefill), for several
// sequences at once.  Token t of a sequence with `base` cached rows attends over rows
// 0 .. base + t as the cache holds them (4 bits), its own row included: the same as one
// decode call per token.
//
// Kernels (stream-ordered):
//   1. q4_pf_angles : (cos, sin) of every token's 32 pairs, f64.
//   2. q4_pf_query  : Q normed, rotated, scaled, as f16 [head][token][256].
//   3. q4_pf_append : K (normed, rotated, f64) and V quantised into the sequences' tiles.
//   4. q4_pf_values : every held row as f16 [kv head][key][256] -- exact -- each sequence
//                     padded with zeros to whole blocks of 128 keys, so that a block never
//                     meets another sequence's values.
//   5. pf_attn      : (pf_attn.cuh) tcgen05 attention, f16 operands: K and V are exact, Q and
//                     P are rounded to 11 bits (bf16's 8 would cost the output's last bits).
#include "pf_attn.cuh"
#include "q4.cuh"

namespace dz {
namespace q4 {

// One launch: sequence i (in the caller's order) has new tokens [row0[i], row0[i + 1]) and
// keys [0, base + T) at K/V rows key0[i]...
struct Prompt {
    int n;
    int32_t sid[MAXB], base[MAXB];
    int32_t row0[MAXB + 1], key0[MAXB + 1];      // key0: multiples of 128
    int32_t at0[MAXB + 1];                       // tiles that the new tokens touch
    __host__ __device__ int T(int i) const { return row0[i + 1] - row0[i]; }
};
__device__ __forceinline__ int last_at_or_before(const int32_t* start, int n, int at) {   // last i with start[i] <= at
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= at) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(256) q4_pf_angles_kernel(const __grid_constant__ Prompt d, RopeAxes axes,
                                                           const int32_t* __restrict__ pos, double2* __restrict__ cs) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / (ROPE / 2)), pair = (int)(i % (ROPE / 2));
    if (t >= d.row0[d.n]) return;
    if (pos) {
        cs[i] = rope_cs(axes, pair, pos[3 * (int64_t)t], pos[3 * (int64_t)t + 1], pos[3 * (int64_t)t + 2]);
    } else {
        const int s = last_at_or_before(d.row0, d.n, t), p = d.base[s] + (t - d.row0[s]);
        cs[i] = rope_cs(axes, pair, p, p, p);
    }
}

__device__ __forceinline__ void load_row(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = tc::bf16_lo_f(w[i]);
        x[2 * i + 1] = tc::bf16_hi_f(w[i]);
    }
}

// one warp per (token, q head)
template <typename T>
__global__ void __launch_bounds__(256) q4_pf_query_kernel(int n_tokens, int nq, const double2* __restrict__ cs,
                                                          const float* __restrict__ q_norm, const T* __restrict__ q_gate,
                                                          __half* __restrict__ q, float eps) {
    const int t = blockIdx.x, head = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= nq) return;
    float x[8];
    load_row(q_gate + ((size_t)t * nq + head) * QG_ROW + 8 * lane, x);
    norm_rotate(x, q_norm, cs + (size_t)t * (ROPE / 2), eps, lane);
    constexpr float QS = 0.0625f * LOG2E;        // scores in log2 units
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pf::pack2<__half>(x[2 * i] * QS, x[2 * i + 1] * QS);
    *reinterpret_cast<uint4*>(q + ((size_t)head * n_tokens + t) * HD + 8 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
}

// one warp per (tile that a new token lies in, kv head); the tile's other positions stay
template <typename T>
__global__ void __launch_bounds__(256) q4_pf_append_kernel(const __grid_constant__ Prompt d, int kvc,
                                                           const Q4Slot* __restrict__ slots,
                                                           const double2* __restrict__ cs,
                                                           const float* __restrict__ k_norm, const T* __restrict__ k,
                                                           const T* __restrict__ v, bool track, float eps) {
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (task >= (int64_t)d.at0[d.n] * kvc) return;
    const int at = (int)(task / kvc), kvh = (int)(task - (int64_t)at * kvc);
    const int s = last_at_or_before(d.at0, d.n, at);
    const int base = d.base[s], end = base + d.T(s);
    const int t16 = (base >> 4) + (at - d.at0[s]);
    const Q4Slot slot = slots[d.sid[s]];
    uint8_t* tile = slot.tile(kvh, t16);
    uint4 w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = *v_words(tile, lane, c);
#pragma unroll
    for (int p = 0; p < Q4_TILE; ++p) {
        const int at_pos = t16 * Q4_TILE + p;
        if (at_pos < base || at_pos >= end) continue;
        const int64_t row = d.row0[s] + (at_pos - base);
        float f[8];
        load_row(k + (row * kvc + kvh) * HD + 8 * lane, f);
        double x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f[e];
        norm_rotate(x, k_norm, cs + row * (ROPE / 2), eps, lane);
        uint32_t code[8];
        uint32_t sb = quantise(x, code);
        put_k(tile, p, lane, code, sb);
        load_row(v + (row * kvc + kvh) * HD + 8 * lane, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f[e];
        sb = quantise(x, code);
        merge_v(w[(p & 7) >> 1], p, code);
        put_v_scale(tile, p, lane, sb);
        if (track && lane == 0) slot.wts[(size_t)kvh * slot.cap + at_pos] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) *v_words(tile, lane, c) = w[c];
}

// one warp per (16 key rows, kv head)
__global__ void __launch_bounds__(256) q4_pf_values_kernel(const __grid_constant__ Prompt d, int kvc,
                                                           const Q4Slot* __restrict__ slots, __half* __restrict__ kf,
                                                           __half* __restrict__ vf) {
    const int64_t keys = d.key0[d.n];
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (task >= keys / Q4_TILE * kvc) return;
    const int kvh = (int)(task % kvc), row = (int)(task / kvc) * Q4_TILE;
    const int s = last_at_or_before(d.key0, d.n, row);
    const int pos = row - d.key0[s], len = d.base[s] + d.T(s);
    const uint8_t* tile = slots[d.sid[s]].tile(kvh, pos >> 4);
    uint4* ko = reinterpret_cast<uint4*>(kf + ((size_t)kvh * keys + row) * HD) + lane;
    uint4* vo = reinterpret_cast<uint4*>(vf + ((size_t)kvh * keys + row) * HD) + lane;
    for (int p = 0; p < Q4_TILE; ++p, ko += HD / 8, vo += HD / 8) {
        uint32_t a[4] = {}, b[4] = {};
        if (pos + p < len) {
            get_k(tile, p, lane, a);
            get_v(tile, p, lane, b);
        }
        *ko = make_uint4(a[0], a[1], a[2], a[3]);
        *vo = make_uint4(b[0], b[1], b[2], b[3]);
    }
}

}  // namespace q4

namespace pf {
// Packed sequences, those with the most keys first and their latest query tiles first: the
// heaviest tiles start first.
struct Packed {
    int n, split_idx, split_cnt;
    int32_t first[MAXB + 1];                     // query tiles before the i-th sequence of this order
    int32_t T[MAXB], base[MAXB], row[MAXB], key[MAXB];
    __host__ __device__ static int own_tiles(int64_t T, int idx, int cnt) {
        const int n_qt = (int)((T + BM - 1) / BM);
        return n_qt > idx ? (n_qt - 1 - idx) / cnt + 1 : 0;
    }
    __device__ __forceinline__ Tile tile(int i) const {
        const int s = q4::last_at_or_before(first, n, i);
        const int own = first[s + 1] - first[s];
        const int64_t q0 = (int64_t)(split_idx + split_cnt * (own - 1 - (i - first[s]))) * BM;
        return {q0, T[s], base[s], row[s] + q0, key[s]};
    }
};
}  // namespace pf

template <typename T>
static cudaError_t launch_group(dz_ctx* ctx, int layer, const q4::Prompt& d, const int32_t* pos, const T* q_gate,
                                const T* k, const T* v, T* out, cudaStream_t st, int* n_launch) {
    const LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
    const int64_t tokens = d.row0[d.n], keys = d.key0[d.n];
    const size_t qn = (size_t)nq * tokens * HD, kn = (size_t)kvc * keys * HD;
    cudaError_t e = ensure_q4_scratch(ctx, (qn + 2 * kn) * sizeof(__half) + (size_t)tokens * (ROPE / 2) * sizeof(double2));
    if (e != cudaSuccess) return e;
    double2* cs = static_cast<double2*>(ctx->q4_scratch);
    __half* qf = reinterpret_cast<__half*>(cs + (size_t)tokens * (ROPE / 2));
    __half *kf = qf + qn, *vf = kf + kn;
    CUtensorMap mq, mk, mv;
    if (!pf::make_map<__half>(&mq, qf, tokens, nq, pf::BM) || !pf::make_map<__half>(&mk, kf, keys, kvc, pf::BN) ||
        !pf::make_map<__half>(&mv, vf, keys, kvc, 32))
        return cudaErrorInvalidValue;
    pf::Packed map;
    map.n = d.n;
    map.split_idx = ctx->cfg.qtile_split_index;
    map.split_cnt = ctx->cfg.qtile_split_count;
    int order[MAXB];
    for (int i = 0; i < d.n; ++i) order[i] = i;
    std::sort(order, order + d.n, [&](int a, int b) {
        const int64_t ka = (int64_t)d.base[a] + d.T(a), kb = (int64_t)d.base[b] + d.T(b);
        return ka != kb ? ka > kb : a < b;
    });
    map.first[0] = 0;
    for (int i = 0; i < d.n; ++i) {
        const int s = order[i];
        map.T[i] = d.T(s);
        map.base[i] = d.base[s];
        map.row[i] = d.row0[s];
        map.key[i] = d.key0[s];
        map.first[i + 1] = map.first[i] + pf::Packed::own_tiles(d.T(s), map.split_idx, map.split_cnt);
    }
    q4::q4_pf_angles_kernel<<<(unsigned)((tokens * (ROPE / 2) + 255) / 256), 256, 0, st>>>(d, ctx->axes, pos, cs);
    q4::q4_pf_query_kernel<T><<<dim3((unsigned)tokens, (nq + 7) / 8), 256, 0, st>>>((int)tokens, nq, cs, L.q_norm, q_gate,
                                                                                 qf, ctx->cfg.rms_eps);
    q4::q4_pf_append_kernel<T><<<(unsigned)(((int64_t)d.at0[d.n] * kvc + 7) / 8), 256, 0, st>>>(
        d, kvc, L.d_q4, cs, L.k_norm, k, v, ctx->q4_track, ctx->cfg.rms_eps);
    q4::q4_pf_values_kernel<<<(unsigned)((keys / Q4_TILE * kvc + 7) / 8), 256, 0, st>>>(d, kvc, L.d_q4, kf, vf);
    *n_launch += 4;
    if (map.first[d.n] > 0) {
        const size_t smem = sizeof(pf::Smem) + 1024;
        auto kernel = pf_attn_kernel<T, T, __half, pf::Packed>;
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess)
            return e;
        kernel<<<(unsigned)(map.first[d.n] * nq), pf::NTHREADS, smem, st>>>(mq, mk, mv, map, kvc, q_gate, out, ctx->d_err);
        *n_launch += 1;
    }
    return cudaGetLastError();
}

// Sequences are taken in groups whose scratch (f16 queries, keys and values) stays below
// this, unless one alone is larger.
static constexpr int64_t GROUP_BYTES = (int64_t)2 << 30;

template <typename T>
static cudaError_t launch_prompts(dz_ctx* ctx, int layer, int n, const int32_t* seq_ids, const int64_t* lens,
                                  const int32_t* pos, const T* q_gate, const T* k, const T* v, T* out, cudaStream_t st,
                                  int* n_launch) {
    LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
    for (int i = 0; i < n;) {
        q4::Prompt d;
        d.n = 0;
        d.row0[0] = d.key0[0] = d.at0[0] = 0;
        int64_t bytes = 0;
        for (; i < n && d.n < MAXB; ++i) {
            const int64_t base = L.len[seq_ids[i]], T_i = lens[i];
            const int64_t keys = (base + T_i + pf::BN - 1) / pf::BN * pf::BN;
            const int64_t more = T_i * (nq * HD * 2 + ROPE / 2 * 16) + keys * kvc * HD * 4;
            if (T_i == 0) continue;
            if (d.n > 0 && bytes + more > GROUP_BYTES) break;
            bytes += more;
            const int s = d.n++;
            d.sid[s] = seq_ids[i];
            d.base[s] = (int32_t)base;
            d.row0[d.n] = d.row0[s] + (int32_t)T_i;
            d.key0[d.n] = d.key0[s] + (int32_t)keys;
            d.at0[d.n] = d.at0[s] + (int32_t)((base + T_i - 1) / Q4_TILE - base / Q4_TILE + 1);
        }
        if (d.n == 0) break;
        const cudaError_t e = launch_group<T>(ctx, layer, d, pos, q_gate, k, v, out, st, n_launch);
        if (e != cudaSuccess) return e;
        const size_t rows = d.row0[d.n];
        for (int s = 0; s < d.n; ++s) L.len[d.sid[s]] += d.T(s);
        if (pos) pos += 3 * rows;
        q_gate += rows * nq * QG_ROW;
        k += rows * kvc * HD;
        v += rows * kvc * HD;
        out += rows * nq * HD;
    }
    return cudaSuccess;
}

cudaError_t launch_q4_prefill(dz_ctx* ctx, int layer, int n, const int32_t* seq_ids, const int64_t* lens,
                              const int32_t* pos, const float* q_gate, const float* k, const float* v, float* out,
                              cudaStream_t st, int* n_launch) {
    return launch_prompts(ctx, layer, n, seq_ids, lens, pos, q_gate, k, v, out, st, n_launch);
}
cudaError_t launch_q4_prefill(dz_ctx* ctx, int layer, int n, const int32_t* seq_ids, const int64_t* lens,
                              const int32_t* pos, const uint16_t* q_gate, const uint16_t* k, const uint16_t* v,
                              uint16_t* out, cudaStream_t st, int* n_launch) {
    using B = __nv_bfloat16;
    return launch_prompts(ctx, layer, n, seq_ids, lens, pos, reinterpret_cast<const B*>(q_gate),
                          reinterpret_cast<const B*>(k), reinterpret_cast<const B*>(v), reinterpret_cast<B*>(out), st,
                          n_launch);
}

}  // namespace dz
