// q4_prefill.cu -- prompts into 4-bit KV caches: packed sequences of different lengths,
// rotary positions of three axes, causal attention over the held rows.
//
// Reference: Daiza-engine/src/model/forward.rs:599-721 (parallel GQA prefill), for several
// sequences at once.  Token t of a sequence with `base` cached rows attends over rows
// 0 .. base + t as the cache holds them (4 bits), its own row included: the same as one
// decode call per token.
//
// Two kernels:
//   1. q4_pf_prep : Q normed, rotated, scaled, as f16 [head][token][256]; K (normed, rotated,
//                   f64) and V quantised into the sequences' tiles; and every held row, old
//                   and new, as f16 [kv head][key][256] -- exact -- each sequence padded with
//                   zeros to whole blocks of 128 keys, so that a block never meets another
//                   sequence's values.  Blocks of three kinds, all independent.
//   2. pf_attn    : (pf_attn.cuh) tcgen05 attention, f16 operands: K and V are exact, Q and P
//                   are rounded to 11 bits (bf16's 8 would cost the output's last bits).
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
    int32_t old0[MAXB + 1];                      // tiles with cached rows or padding
    __host__ __device__ int T(int i) const { return row0[i + 1] - row0[i]; }
    // tiles of cached rows come first, then those of the padding
    __host__ __device__ int cached_tiles(int i) const { return (base[i] + Q4_TILE - 1) / Q4_TILE; }
    __host__ __device__ int first_pad_tile(int i) const { return (base[i] + T(i)) / Q4_TILE; }
};
__device__ __forceinline__ int last_at_or_before(const int32_t* start, int n, int at) {   // last i with start[i] <= at
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= at) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ void load_row(const T* p, double (&x)[8]) {
    const float4 a = as_f32(load4(p)), b = as_f32(load4(p + 4));
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
// codes + 8 and the group's scale byte -> 8 held values
__device__ __forceinline__ uint4 held(const uint32_t (&code)[8], uint32_t sb) {
    const uint32_t s = scale_pair(sb | sb << 16), c = hmul2_u(s, NEG72);
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = unpack(code[2 * i] << 4 | code[2 * i + 1] << 20, s, c);
    return make_uint4(h[0], h[1], h[2], h[3]);
}

constexpr int PREP_WARPS = 16, PREP_HEADS = 6;   // heads of a token that a warp takes

// Blocks [0, at0 kvc): a tile of new rows and a kv head, a warp per position.
// Then (old0 kvc) blocks: a tile of cached rows or padding, a warp per position.
// Then: a warp per (token, PREP_HEADS heads).
template <typename T>
__global__ void __launch_bounds__(32 * PREP_WARPS)
    q4_pf_prep_kernel(const __grid_constant__ Prompt d, const __grid_constant__ RopeAxes axes, int kvc,
                      const Q4Slot* __restrict__ slots, const int32_t* __restrict__ pos, const float* __restrict__ q_norm,
                      const float* __restrict__ k_norm, const T* __restrict__ q_gate, const T* __restrict__ k,
                      const T* __restrict__ v, __half* __restrict__ qf, __half* __restrict__ kf, __half* __restrict__ vf,
                      bool track, float eps) {
    __shared__ TileMerge merge;
    __shared__ double2 cs[PREP_WARPS][ROPE / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nq = GRP * kvc;
    const int64_t keys = d.key0[d.n], tokens = d.row0[d.n];
    int64_t block = blockIdx.x;
    auto angles_at = [&](int s, int64_t row, int (&p)[3]) {
        if (pos) {
            for (int i = 0; i < 3; ++i) p[i] = pos[3 * row + i];
        } else {
            p[0] = p[1] = p[2] = d.base[s] + (int)(row - d.row0[s]);
        }
    };
    if (block < (int64_t)d.at0[d.n] * kvc) {
        const int at = (int)(block / kvc), kvh = (int)(block - (int64_t)at * kvc);
        const int s = last_at_or_before(d.at0, d.n, at);
        const int base = d.base[s], t16 = (base >> 4) + (at - d.at0[s]), slot_pos = t16 * Q4_TILE + warp;
        const Q4Slot slot = slots[d.sid[s]];
        uint8_t* tile = slot.tile(kvh, t16);
        merge.begin();
        if (slot_pos >= base && slot_pos < base + d.T(s)) {
            const int64_t row = d.row0[s] + (slot_pos - base);
            int p[3];
            angles_at(s, row, p);
            cs[warp][lane] = rope_cs(axes, lane, p[0], p[1], p[2]);
            __syncwarp();
            const size_t out = ((size_t)kvh * keys + d.key0[s] + slot_pos) * HD + 8 * lane;
            double x[8];
            load_row(k + (row * kvc + kvh) * HD + 8 * lane, x);
            norm_rotate(x, k_norm, cs[warp], eps, lane);
            uint32_t code[8];
            uint32_t sb = quantise(x, code);
            put_k(tile, warp, lane, code, sb);
            *reinterpret_cast<uint4*>(kf + out) = held(code, sb);
            load_row(v + (row * kvc + kvh) * HD + 8 * lane, x);
            sb = quantise(x, code);
            merge.add(warp, lane, code);
            put_v_scale(tile, warp, lane, sb);
            *reinterpret_cast<uint4*>(vf + out) = held(code, sb);
            if (track && lane == 0) slot.wts[(size_t)kvh * slot.cap + slot_pos] = 0.0f;
        }
        merge.end(tile);
        return;
    }
    block -= (int64_t)d.at0[d.n] * kvc;
    if (block < (int64_t)d.old0[d.n] * kvc) {
        const int ot = (int)(block / kvc), kvh = (int)(block - (int64_t)ot * kvc);
        const int s = last_at_or_before(d.old0, d.n, ot);
        const int i = ot - d.old0[s], cached = d.cached_tiles(s);
        const int t16 = i < cached ? i : d.first_pad_tile(s) + (i - cached), at = t16 * Q4_TILE + warp;
        const bool old = i < cached;
        if (old ? at >= d.base[s] : at < d.base[s] + d.T(s)) return;   // a new row
        uint32_t a[4] = {}, b[4] = {};
        if (old) {
            const uint8_t* tile = slots[d.sid[s]].tile(kvh, t16);
            get_k(tile, warp, lane, a);
            get_v(tile, warp, lane, b);
        }
        const size_t out = ((size_t)kvh * keys + d.key0[s] + at) * HD + 8 * lane;
        *reinterpret_cast<uint4*>(kf + out) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(vf + out) = make_uint4(b[0], b[1], b[2], b[3]);
        return;
    }
    block -= (int64_t)d.old0[d.n] * kvc;
    const int parts = (nq + PREP_HEADS - 1) / PREP_HEADS;
    const int64_t task = block * PREP_WARPS + warp, row = task / parts;
    if (row >= tokens) return;
    const int h0 = (int)(task - row * parts) * PREP_HEADS, h1 = min(nq, h0 + PREP_HEADS);
    int p[3];
    angles_at(pos ? 0 : last_at_or_before(d.row0, d.n, (int)row), row, p);
    float2 c4[4];
    spread_pairs(rope_cs_f32(axes, lane, p[0], p[1], p[2]), c4, lane);
    float w[8];
    load_split(q_norm, lane, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] *= 0.0625f * LOG2E;   // scores in log2 units
    SplitRow<T> in[PREP_HEADS];
#pragma unroll
    for (int i = 0; i < PREP_HEADS; ++i)
        if (h0 + i < h1) in[i].load(q_gate + (row * nq + h0 + i) * QG_ROW, lane);
#pragma unroll
    for (int i = 0; i < PREP_HEADS; ++i) {
        if (h0 + i >= h1) break;
        float x[8];
        in[i].values(x);
        norm_rotate_split(x, w, c4, eps, lane);
        __half* out = qf + ((size_t)(h0 + i) * tokens + row) * HD;
        *reinterpret_cast<uint2*>(out + split_dim(lane, 0)) =
            make_uint2(pf::pack2<__half>(x[0], x[1]), pf::pack2<__half>(x[2], x[3]));
        *reinterpret_cast<uint2*>(out + split_dim(lane, 1)) =
            make_uint2(pf::pack2<__half>(x[4], x[5]), pf::pack2<__half>(x[6], x[7]));
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
    cudaError_t e = ensure_q4_scratch(ctx, (qn + 2 * kn) * sizeof(__half));
    if (e != cudaSuccess) return e;
    __half* qf = static_cast<__half*>(ctx->q4_scratch);
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
    const int64_t q_tasks = tokens * ((nq + q4::PREP_HEADS - 1) / q4::PREP_HEADS);
    const int64_t blocks = (int64_t)(d.at0[d.n] + d.old0[d.n]) * kvc + (q_tasks + q4::PREP_WARPS - 1) / q4::PREP_WARPS;
    q4::q4_pf_prep_kernel<T><<<(unsigned)blocks, 32 * q4::PREP_WARPS, 0, st>>>(
        d, ctx->axes, kvc, L.d_q4, pos, L.q_norm, L.k_norm, q_gate, k, v, qf, kf, vf, ctx->q4_track, ctx->cfg.rms_eps);
    *n_launch += 1;
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
        d.row0[0] = d.key0[0] = d.at0[0] = d.old0[0] = 0;
        int64_t bytes = 0;
        for (; i < n && d.n < MAXB; ++i) {
            const int64_t base = L.len[seq_ids[i]], T_i = lens[i];
            const int64_t keys = (base + T_i + pf::BN - 1) / pf::BN * pf::BN;
            const int64_t more = T_i * nq * HD * 2 + keys * kvc * HD * 4;
            if (T_i == 0) continue;
            if (d.n > 0 && bytes + more > GROUP_BYTES) break;
            bytes += more;
            const int s = d.n++;
            d.sid[s] = seq_ids[i];
            d.base[s] = (int32_t)base;
            d.row0[d.n] = d.row0[s] + (int32_t)T_i;
            d.key0[d.n] = d.key0[s] + (int32_t)keys;
            d.at0[d.n] = d.at0[s] + (int32_t)((base + T_i - 1) / Q4_TILE - base / Q4_TILE + 1);
            d.old0[d.n] = d.old0[s] + d.cached_tiles(s) + (int32_t)(keys / Q4_TILE - d.first_pad_tile(s));
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
