// q4_decode.cu -- split-K decode attention over the 4-bit KV cache (q4.cuh).
//
// The gated GQA core of attention.rs:90-203 for one token per sequence, with K and V
// held in 4 bits and rotary positions of three axes.  Stream-ordered kernels:
//   1. q4_prep     : per sequence and head -- deinterleave [Q_h | gate_h], QK-RMSNorm,
//                    rotation; q as matrix operand, K and V quantised into slot len.
//   2. q4_split    : per (sequence, chunk, kv head), one warp each: scores, online
//                    softmax, P V over the chunk's tiles; unnormalised partials out.
//   3. gqa_combine : (gqa_decode.cu) merge, normalise, gate.
//   4. q4_weights  : tracked caches -- the new attention weights are added.
#include <algorithm>
#include <cstddef>

#include "q4.cuh"

namespace dz {
namespace q4 {

// ---------------------------------------------------------------------------
// 1. prep: grid (B, ceil((nq + kvc) / 8)), one head per warp.
//    q is scaled by log2(e) / 16 (scores in log2 units) and by a power of two that
//    puts the head's largest magnitude into [2^11, 2^12), then split into f16 hi + lo
//    (22 bits; f16 subnormals start 2^25 below), in the register order of the A
//    operand of mma.m16n8k16: rows 0..7 are the hi parts of the group's heads (6 and 7
//    empty), rows 8..15 the lo parts, so one product of K gives both.
//      q_frag [b][kvh][step 16][lane][hi 0,1 | lo 0,1 | hi 2,3 | lo 2,3]
//    where step s, lane (r, c) covers dims 64 c + 4 s .. + 3 of head r.
// ---------------------------------------------------------------------------
constexpr int FRAG_WORDS = 16 * 32 * 4;       // words of q_frag per (sequence, kv head)

__global__ void __launch_bounds__(256) q4_prep_kernel(GqaDecodeDesc d, Q4Pos pos, RopeAxes axes, int kvc,
                                                      const Q4Slot* __restrict__ slots,
                                                      const float* __restrict__ q_norm, const float* __restrict__ k_norm,
                                                      const float* __restrict__ q_gate, const float* __restrict__ k_in,
                                                      const float* __restrict__ v_in, uint32_t* __restrict__ q_frag,
                                                      float* __restrict__ q_scale, float eps) {
    __shared__ double2 cs[ROPE / 2];
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) cs[lane] = rope_cs(axes, lane, pos.p[b][0], pos.p[b][1], pos.p[b][2]);
    __syncthreads();
    // As in gqa_prep: everything before this grid is complete (inputs, caches, q_frag)
    // before the split grid may start streaming old tiles.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int nq = GRP * kvc;
    const int task = blockIdx.y * 8 + warp;
    if (task >= nq + kvc) return;
    if (task < nq) {
        const float4* src = reinterpret_cast<const float4*>(q_gate + ((size_t)b * nq + task) * QG_ROW);
        const float4 a0 = src[2 * lane], a1 = src[2 * lane + 1];
        float x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
        norm_rotate(x, q_norm, cs, eps, lane);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] *= 0.0625f * LOG2E;
            amax = fmaxf(amax, fabsf(x[e]));
        }
        amax = warp_max(amax);
        const int ex = (int)(__float_as_uint(amax) >> 23);
        const int field = min(max(265 - ex, 1), 253);          // exponent field of 2^(11 - exponent of amax)
        const float up = __uint_as_float((uint32_t)field << 23);
        const int kvh = task / GRP, r = task - kvh * GRP;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float u = x[2 * i] * up, w = x[2 * i + 1] * up;
            const __half2 h = __floats2half2_rn(u, w);
            const __half2 l = __floats2half2_rn(u - __low2float(h), w - __high2float(h));
            hi[i] = *reinterpret_cast<const uint32_t*>(&h);
            lo[i] = *reinterpret_cast<const uint32_t*>(&l);
        }
        uint4* dst = reinterpret_cast<uint4*>(q_frag + (size_t)(b * kvc + kvh) * FRAG_WORDS);
        const int at = (lane & 7) * 64 + r * 4 + (lane >> 3);  // steps 2 w and 2 w + 1 of word w = lane % 8, c = lane / 8
        dst[at] = make_uint4(hi[0], lo[0], hi[1], lo[1]);
        dst[at + 32] = make_uint4(hi[2], lo[2], hi[3], lo[3]);
        if (lane == 0)
            q_scale[(b * kvc + kvh) * 8 + r] = __uint_as_float((uint32_t)(254 - field) << 23);
    } else {
        const int kvh = task - nq, slot_pos = d.len[b];
        uint4* dst = reinterpret_cast<uint4*>(q_frag + (size_t)(b * kvc + kvh) * FRAG_WORDS);
#pragma unroll
        for (int i = 0; i < 4; ++i)                            // the operand's empty rows: heads 6 and 7
            dst[(4 * i + (lane >> 3)) * 32 + 24 + (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
        if (lane < 2) q_scale[(b * kvc + kvh) * 8 + 6 + lane] = 0.0f;
        uint8_t* tile = slots[d.sid[b]].tile(kvh, slot_pos >> 4);
        const int p = slot_pos & 15;
        const size_t at = ((size_t)b * kvc + kvh) * HD + 8 * lane;
        const float4 k0 = *reinterpret_cast<const float4*>(k_in + at), k1 = *reinterpret_cast<const float4*>(k_in + at + 4);
        const float4 v0 = *reinterpret_cast<const float4*>(v_in + at), v1 = *reinterpret_cast<const float4*>(v_in + at + 4);
        double x[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
        norm_rotate(x, k_norm, cs, eps, lane);
        uint32_t code[8];
        uint32_t sb = quantise(x, code);
        put_k(tile, p, lane, code, sb);
        double y[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        sb = quantise(y, code);
        uint4* vw = v_words(tile, lane, (p & 7) >> 1);
        uint4 w = *vw;
        merge_v(w, p, code);
        *vw = w;
        put_v_scale(tile, p, lane, sb);
    }
}

// ---------------------------------------------------------------------------
// 2. split-K attention, one warp per (sequence, chunk, kv head).
//    A tile (16 positions, 4352 bytes) is one bulk copy into the warp's own ring.
//    Scores: S = Q K^T, A = q (hi rows, lo rows), B = the 8 positions of a K word row,
//    16 steps of 16 dims; thread (r, c) gets head r at positions 2c, 2c+1 (hi sum and
//    lo sum, added).  That is the B operand's own layout, so P needs no shuffle:
//    O^T += V^T P^T, A = V's dims x 16 positions, B = P (hi, then lo), 16 tiles of 16
//    dims accumulated in 64 registers.
// ---------------------------------------------------------------------------
constexpr int Q4_STAGES = 4;
constexpr int Q4_WARPS = GQA_SPLIT_WARPS;
constexpr float P_LOG2 = 12.0f;               // p is scaled by 2^12: its f16 lo part keeps 11 bits down to 2^-11

struct alignas(128) Q4Ring {
    uint8_t tile[Q4_STAGES][Q4_TILE_BYTES];
    uint64_t full[Q4_STAGES];
};
static_assert(sizeof(Q4Ring) % 128 == 0 && Q4_TILE_BYTES % 128 == 0, "bulk copies need 16-byte alignment");
struct Q4Smem { Q4Ring w[Q4_WARPS]; };

struct Q4Item { int b, kvh, p0, p1, ntiles; const uint8_t* base; };

__device__ __forceinline__ Q4Item q4_item(const GqaDecodeDesc& d, int kvc, const Q4Slot* __restrict__ slots, int item) {
    Q4Item it;
    const int chunk_idx = item / kvc;
    it.kvh = item - chunk_idx * kvc;
    int lo = 0, hi = d.B - 1;                    // last b with cum[b] <= chunk_idx
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (d.cum[mid] <= chunk_idx) lo = mid; else hi = mid - 1;
    }
    it.b = lo;
    it.p0 = (chunk_idx - d.cum[lo]) * d.chunk;   // a multiple of 16
    it.p1 = min(d.len[lo] + 1, it.p0 + d.chunk);
    it.ntiles = (it.p1 - it.p0 + Q4_TILE - 1) / Q4_TILE;
    it.base = slots[d.sid[lo]].tile(it.kvh, it.p0 >> 4);
    return it;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool TRACK>
__global__ void __launch_bounds__(32 * Q4_WARPS, 1)
    q4_split_kernel(GqaDecodeDesc d, int kvc, const Q4Slot* __restrict__ slots, const uint32_t* __restrict__ q_frag,
                    const float* __restrict__ q_scale, float* __restrict__ part_o, float* __restrict__ part_ml,
                    float* __restrict__ scores, int* err, int n_items) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Q4Ring& R = reinterpret_cast<Q4Smem*>(smem_raw)->w[threadIdx.x >> 5];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int gw = blockIdx.x * Q4_WARPS + warp, nw = gridDim.x * Q4_WARPS;
    if (lane == 0) {
        for (int s = 0; s < Q4_STAGES; ++s) mbar_init(&R.full[s], 1);
        fence_mbar_init();
    }
    __syncwarp();
    asm volatile("griddepcontrol.launch_dependents;");
    int p_item = gw, p_tile = 0;
    Q4Item pinfo{};
    if (p_item < n_items) pinfo = q4_item(d, kvc, slots, p_item);
    // the tile that holds slot len is written by q4_prep: requested after the grid-dependency wait
    bool dep_done = false;
    auto wait_prep = [&]() {
        if (!dep_done) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            dep_done = true;
        }
    };
    auto produce = [&](int stage) {
        if (p_item >= n_items) return;
        if (pinfo.p0 + (p_tile + 1) * Q4_TILE > d.len[pinfo.b]) wait_prep();
        if (lane == 0) {
            mbar_arrive_expect_tx(&R.full[stage], Q4_TILE_BYTES);
            bulk_g2s(R.tile[stage], pinfo.base + (size_t)p_tile * Q4_TILE_BYTES, Q4_TILE_BYTES, &R.full[stage]);
        }
        if (++p_tile == pinfo.ntiles) {
            p_item += nw;
            p_tile = 0;
            if (p_item < n_items) pinfo = q4_item(d, kvc, slots, p_item);
        }
    };
    for (int s = 0; s < Q4_STAGES; ++s) produce(s);
    wait_prep();                                 // q_frag

    int j = 0;
    for (int item = gw; item < n_items; item += nw) {
        const Q4Item it = q4_item(d, kvc, slots, item);
        uint4 q[16];
        {
            const uint4* src = reinterpret_cast<const uint4*>(q_frag + (size_t)(it.b * kvc + it.kvh) * FRAG_WORDS) + lane;
#pragma unroll
            for (int s = 0; s < 16; ++s) q[s] = src[s * 32];
        }
        const float qs = q_scale[(it.b * kvc + it.kvh) * 8 + r];
        float o[16][4];
#pragma unroll
        for (int m = 0; m < 16; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][e] = 0.0f;
        float m_run = -INFINITY, l_run = 0.0f;   // head r; l is this thread's share

        for (int t = 0; t < it.ntiles; ++t, ++j) {
            const int stage = j % Q4_STAGES;
            if (!mbar_wait(&R.full[stage], (uint32_t)((j / Q4_STAGES) & 1), err)) return;
            const uint8_t* tile = R.tile[stage];
            // ---- scores of 2 x 8 positions
            float x[4];
            {
                const uint32_t kb = *reinterpret_cast<const uint32_t*>(tile + OFF_KS + lane * 4);
#pragma unroll
                for (int n8 = 0; n8 < 2; ++n8) {
                    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 w4 = *reinterpret_cast<const uint4*>(tile + (n8 * 2 + i) * 512 + lane * 16);
                        // the group's scale byte in both halves
                        const uint32_t sc = scale_pair(__byte_perm(kb, 0u, 0x4040 + 0x0101 * (n8 * 2 + i)));
                        const uint32_t cc = hmul2_u(sc, NEG72);
                        const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const uint32_t w = ws[u];
                            const uint4 qa = q[8 * i + 2 * u], qb = q[8 * i + 2 * u + 1];
                            mma(s0, qa.x, qa.y, qa.z, qa.w, unpack(w << 4, sc, cc), unpack(w, sc, cc));
                            mma(s1, qb.x, qb.y, qb.z, qb.w, unpack(w >> 4, sc, cc), unpack(w >> 8, sc, cc));
                        }
                    }
                    x[2 * n8] = ((s0[0] + s1[0]) + (s0[2] + s1[2])) * qs;
                    x[2 * n8 + 1] = ((s0[1] + s1[1]) + (s0[3] + s1[3])) * qs;
                }
            }
            const int pos = it.p0 + t * Q4_TILE + 2 * c;
            if (TRACK) {
                if (r < GRP) {
                    // [tile of the launch][kvh][head][16]; tiles of sequence b start at tile_cum
                    float* sc = scores + (((size_t)d.pos[it.b] + ((it.p0 >> 4) + t)) * kvc + it.kvh) * (GRP * Q4_TILE) +
                                r * Q4_TILE + 2 * c;
                    *reinterpret_cast<float2*>(sc) = make_float2(x[0], x[1]);
                    *reinterpret_cast<float2*>(sc + 8) = make_float2(x[2], x[3]);
                }
            }
            if (t == it.ntiles - 1) {
                if (pos >= it.p1) x[0] = -INFINITY;
                if (pos + 1 >= it.p1) x[1] = -INFINITY;
                if (pos + 8 >= it.p1) x[2] = -INFINITY;
                if (pos + 9 >= it.p1) x[3] = -INFINITY;
            }
            // ---- online softmax
            float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run, mx);
            if (__any_sync(0xffffffffu, m_new > m_run)) {
                const float a = ex2f(m_run - m_new);
                l_run *= a;
                const float a0 = __shfl_sync(0xffffffffu, a, 8 * c), a1 = __shfl_sync(0xffffffffu, a, 8 * c + 4);
#pragma unroll
                for (int m = 0; m < 16; ++m) {
                    o[m][0] *= a0;
                    o[m][1] *= a1;
                    o[m][2] *= a0;
                    o[m][3] *= a1;
                }
                m_run = m_new;
            }
            const float off = P_LOG2 - m_run;
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = ex2f(x[e] + off);
                l_run += p[e];
            }
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2 h = __floats2half2_rn(p[2 * i], p[2 * i + 1]);
                const __half2 l = __floats2half2_rn(p[2 * i] - __low2float(h), p[2 * i + 1] - __high2float(h));
                ph[i] = *reinterpret_cast<const uint32_t*>(&h);
                pl[i] = *reinterpret_cast<const uint32_t*>(&l);
            }
            // ---- O^T += V^T P^T
            {
                const uint32_t vb = *reinterpret_cast<const uint32_t*>(tile + OFF_VS + lane * 4);
                const uint32_t sa = scale_pair(__byte_perm(vb, 0u, 0x4140)), sb = scale_pair(__byte_perm(vb, 0u, 0x4342));
                const uint32_t ca = hmul2_u(sa, NEG72), cb = hmul2_u(sb, NEG72);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(tile + OFF_V + i * 512 + lane * 16);
                    const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t w = ws[u];
                        const uint32_t a0 = unpack(w << 4, sa, ca), a2 = unpack(w, sb, cb);
                        const uint32_t a1 = unpack(w >> 4, sa, ca), a3 = unpack(w >> 8, sb, cb);
                        mma(o[4 * i + u], a0, a1, a2, a3, ph[0], ph[1]);
                        mma(o[4 * i + u], a0, a1, a2, a3, pl[0], pl[1]);
                    }
                }
            }
            __syncwarp();
            produce(stage);
        }
        // ---- partials: thread (r, c) holds dims 32 r .. + 31 of heads 2c, 2c + 1
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
        if (c < GRP / 2) {
            float* po = part_o + ((size_t)item * GRP + 2 * c) * HD + 32 * r;
#pragma unroll
            for (int m = 0; m < 16; m += 2) {
                *reinterpret_cast<float4*>(po + 2 * m) = make_float4(o[m][0], o[m][2], o[m + 1][0], o[m + 1][2]);
                *reinterpret_cast<float4*>(po + HD + 2 * m) = make_float4(o[m][1], o[m][3], o[m + 1][1], o[m + 1][3]);
            }
        }
        if (c == 0 && r < GRP) {
            part_ml[((size_t)item * GRP + r) * 2 + 0] = m_run - P_LOG2;
            part_ml[((size_t)item * GRP + r) * 2 + 1] = l_run;
        }
    }
}

// ---------------------------------------------------------------------------
// 4. tracked caches: weight of position j of a kv head += sum over its 6 q heads of
//    exp2(score - M) / L, with M and L merged from the chunks' (m, l).  The new
//    position's weight starts here.  Grid (ceil(longest / 1024), kvc, B).
// ---------------------------------------------------------------------------
constexpr int WT_SPAN = 1024;

__global__ void __launch_bounds__(256) q4_weights_kernel(GqaDecodeDesc d, int kvc, const Q4Slot* __restrict__ slots,
                                                         const float* __restrict__ part_ml,
                                                         const float* __restrict__ scores) {
    __shared__ float M[GRP], L[GRP];
    const int b = blockIdx.z, kvh = blockIdx.y, n = d.len[b] + 1, j0 = blockIdx.x * WT_SPAN;
    if (j0 >= n) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < GRP) {
        const int c0 = d.cum[b], nc = d.cum[b + 1] - c0;
        const float2* ml = reinterpret_cast<const float2*>(part_ml) + ((size_t)c0 * kvc + kvh) * GRP + warp;
        float m = -INFINITY;
        for (int i = lane; i < nc; i += 32) m = fmaxf(m, ml[(size_t)i * kvc * GRP].x);
        m = warp_max(m);
        float l = 0.0f;
        for (int i = lane; i < nc; i += 32) {
            const float2 v = ml[(size_t)i * kvc * GRP];
            l += v.y * exp2f(v.x - m);
        }
        l = warp_sum(l);
        if (lane == 0) {
            M[warp] = m;
            L[warp] = 1.0f / l;
        }
    }
    __syncthreads();
    const Q4Slot slot = slots[d.sid[b]];
    float* wts = slot.wts + (size_t)kvh * slot.cap;
    for (int j = j0 + threadIdx.x; j < min(n, j0 + WT_SPAN); j += 256) {
        const float* sc = scores + (((size_t)d.pos[b] + (j >> 4)) * kvc + kvh) * (GRP * Q4_TILE) + (j & 15);
        float w = 0.0f;
#pragma unroll
        for (int h = 0; h < GRP; ++h) w += ex2f(sc[h * Q4_TILE] - M[h]) * L[h];
        wts[j] = w + (j < n - 1 ? wts[j] : 0.0f);
    }
}

}  // namespace q4

cudaError_t launch_q4_decode(dz_ctx* ctx, int layer, const GqaDecodeDesc& d, const Q4Pos& pos, const float* q_gate,
                             const float* k, const float* v, float* out, cudaStream_t st, int* n_launch) {
    using namespace q4;
    const LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count;
    const int items = d.cum[d.B] * kvc;
    auto split = ctx->q4_track ? q4_split_kernel<true> : q4_split_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(split, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Q4Smem));
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(d.B, (GRP * kvc + kvc + 7) / 8);
    lc.blockDim = dim3(256);
    lc.stream = st;
    lc.attrs = at;
    lc.numAttrs = 1;
    e = cudaLaunchKernelEx(&lc, q4_prep_kernel, d, pos, ctx->axes, kvc, (const Q4Slot*)L.d_q4, (const float*)L.q_norm,
                           (const float*)L.k_norm, q_gate, k, v, ctx->q4_frag, ctx->q4_qs, ctx->cfg.rms_eps);
    if (e != cudaSuccess) return e;
    lc.gridDim = dim3(std::min((items + Q4_WARPS - 1) / Q4_WARPS, ctx->n_sm));
    lc.blockDim = dim3(32 * Q4_WARPS);
    lc.dynamicSmemBytes = sizeof(Q4Smem);
    e = cudaLaunchKernelEx(&lc, split, d, kvc, (const Q4Slot*)L.d_q4, (const uint32_t*)ctx->q4_frag,
                           (const float*)ctx->q4_qs, ctx->part_o, ctx->part_ml, ctx->q4_sc, ctx->d_err, items);
    if (e != cudaSuccess) return e;
    if ((e = launch_gqa_combine(ctx, d, q_gate, out, st, ctx->part_o, ctx->part_ml)) != cudaSuccess) return e;
    *n_launch += 3;
    if (ctx->q4_track) {
        int longest = 0;
        for (int b = 0; b < d.B; ++b) longest = std::max(longest, d.len[b] + 1);
        q4_weights_kernel<<<dim3((longest + WT_SPAN - 1) / WT_SPAN, kvc, d.B), 256, 0, st>>>(
            d, kvc, (const Q4Slot*)L.d_q4, ctx->part_ml, ctx->q4_sc);
        *n_launch += 1;
    }
    return cudaGetLastError();
}

}  // namespace dz
