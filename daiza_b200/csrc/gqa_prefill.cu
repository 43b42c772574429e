// gqa_prefill.cu -- causal GQA prefill: TMA-fed tcgen05/TMEM flash attention.
//
// Reference: Daiza-engine/src/model/forward.rs:599-721 (parallel GQA prefill):
// K-norm + RoPE + append for every token first, then each token t attends over
// base_len + t + 1 cached positions with Q-norm/RoPE/scale applied to its q,
// and the output is multiplied by sigmoid(gate).
//
// Kernels (stream-ordered):
//   1. pf_prep      : per token -- QK-RMSNorm, partial RoPE ('+' sign), q *= 1/16;
//                     writes Q as bf16 [head][T][256], appends K (normed, roped) and
//                     V to the f32 KV cache and to bf16 copies [kvh][len][256].
//   2. pf_prior     : (only when the cache already held tokens) bf16 copies of the
//                     prior K/V rows for the attention kernel.
//   3. pf_attn      : (pf_attn.cuh) one CTA per (q head, 128-token query tile), heaviest tiles
//                     first.  Warp 8 issues TMA loads (Q once; K blocks of 128 keys
//                     as 16 KB 64-dim boxes through a 5-slot ring, V as 16 KB
//                     32-key slots through a 4-slot ring, all 128B-swizzled), warp 9
//                     issues tcgen05.mma from a single thread: S = Q K^T (M128 N128
//                     K256, both operands K-major in SMEM) into one of two TMEM S
//                     buffers, and O += P V (M128 N256 K128, P from TMEM, V MN-major
//                     in SMEM) into a 256-column TMEM accumulator.  Warps 0-7 (one
//                     TMEM lane per query row, two warps per lane quarter splitting
//                     the 128 keys of a block) run the causal online softmax in log2 units
//                     with a lazy rescale of O (only when the row max grows by more
//                     than 2^8), write P as bf16 over its S columns in TMEM, and finish with
//                     O / l * sigmoid(gate).
// All mbarrier waits are bounded (device error word on expiry).
#include "pf_attn.cuh"

namespace dz {

// ---------------------------------------------------------------------------
// 1. prep: per token (blockIdx.x), 8 warps over 6*kvc q heads and kvc kv heads
// ---------------------------------------------------------------------------
template <typename Tin>
__global__ void __launch_bounds__(256) pf_prep_kernel(int kvc, int64_t T, int64_t base, int64_t rope_pos0, KvSlot slot,
                                                      const float* __restrict__ q_norm,
                                                      const float* __restrict__ k_norm,
                                                      const float* __restrict__ rope, const Tin* __restrict__ q_gate,
                                                      const Tin* __restrict__ k_in, const Tin* __restrict__ v_in,
                                                      __nv_bfloat16* __restrict__ qb, __nv_bfloat16* __restrict__ kb,
                                                      __nv_bfloat16* __restrict__ vb, int64_t L, float eps) {
    const int64_t t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nq = GRP * kvc;
    const int64_t pos = base + t;                                   // cache slot
    const float* cs = rope + (rope_pos0 + t) * (2 * ROPE);           // RoPE row of start_pos + t (forward.rs:550-557)
    for (int task = warp; task < nq + kvc; task += 8) {
        const Tin* src;
        const float* w;
        if (task < nq) {
            src = q_gate + (t * nq + task) * QG_ROW;
            w = q_norm;
        } else {
            const int h = task - nq;
            src = k_in + (t * kvc + h) * HD;
            w = k_norm;
            const Tin* vs = v_in + (t * kvc + h) * HD;
            const float4 v0 = ld4<Tin>(vs + 4 * lane), v1 = ld4<Tin>(vs + 128 + 4 * lane);
            float* vd = slot.v + ((size_t)h * slot.cap + pos) * HD;
            reinterpret_cast<float4*>(vd)[lane] = v0;
            reinterpret_cast<float4*>(vd + 128)[lane] = v1;
            __nv_bfloat16* vbd = vb + ((size_t)h * L + pos) * HD;
            st4_bf16(vbd + 4 * lane, v0);
            st4_bf16(vbd + 128 + 4 * lane, v1);
        }
        float4 x0 = ld4<Tin>(src + 4 * lane);
        float4 x1 = ld4<Tin>(src + 128 + 4 * lane);
        float ss = x0.x * x0.x + x0.y * x0.y + x0.z * x0.z + x0.w * x0.w + x1.x * x1.x + x1.y * x1.y +
                   x1.z * x1.z + x1.w * x1.w;
        ss = warp_sum(ss);
        const float inv = 1.0f / sqrtf(ss / (float)HD + eps);
        const float4 w0 = reinterpret_cast<const float4*>(w)[lane];
        const float4 w1 = reinterpret_cast<const float4*>(w)[lane + 32];
        x0 = make_float4((x0.x * inv) * w0.x, (x0.y * inv) * w0.y, (x0.z * inv) * w0.z, (x0.w * inv) * w0.w);
        x1 = make_float4((x1.x * inv) * w1.x, (x1.y * inv) * w1.y, (x1.z * inv) * w1.z, (x1.w * inv) * w1.w);
        float4 pr;
        pr.x = __shfl_xor_sync(0xffffffffu, x0.x, 8);
        pr.y = __shfl_xor_sync(0xffffffffu, x0.y, 8);
        pr.z = __shfl_xor_sync(0xffffffffu, x0.z, 8);
        pr.w = __shfl_xor_sync(0xffffffffu, x0.w, 8);
        if (lane < 16) {
            const float4 c = reinterpret_cast<const float4*>(cs)[lane];
            const float4 s = reinterpret_cast<const float4*>(cs + ROPE)[lane];
            x0 = make_float4(fmaf(x0.x, c.x, pr.x * s.x), fmaf(x0.y, c.y, pr.y * s.y), fmaf(x0.z, c.z, pr.z * s.z),
                             fmaf(x0.w, c.w, pr.w * s.w));
        }
        if (task < nq) {
            // 1/sqrt(256) and log2(e): the attention kernel's scores come out in log2 units
            constexpr float QS = 0.0625f * 1.4426950408889634f;
            x0 = make_float4(x0.x * QS, x0.y * QS, x0.z * QS, x0.w * QS);
            x1 = make_float4(x1.x * QS, x1.y * QS, x1.z * QS, x1.w * QS);
            __nv_bfloat16* qd = qb + ((size_t)task * T + t) * HD;
            st4_bf16(qd + 4 * lane, x0);
            st4_bf16(qd + 128 + 4 * lane, x1);
        } else {
            const int h = task - nq;
            float* kd = slot.k + ((size_t)h * slot.cap + pos) * HD;
            reinterpret_cast<float4*>(kd)[lane] = x0;
            reinterpret_cast<float4*>(kd + 128)[lane] = x1;
            __nv_bfloat16* kbd = kb + ((size_t)h * L + pos) * HD;
            st4_bf16(kbd + 4 * lane, x0);
            st4_bf16(kbd + 128 + 4 * lane, x1);
        }
    }
}

// 2. bf16 copies of rows [0, base) of the f32 cache
__global__ void pf_prior_kernel(int kvc, int64_t base, KvSlot slot, __nv_bfloat16* __restrict__ kb,
                                __nv_bfloat16* __restrict__ vb, int64_t L) {
    const int64_t n4 = (int64_t)kvc * base * (HD / 4);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n4; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t e = i * 4;
        const int64_t h = e / (base * HD);
        const int64_t r = e - h * base * HD;     // row * HD + d
        const float4 kx = *reinterpret_cast<const float4*>(slot.k + (size_t)h * slot.cap * HD + r);
        const float4 vx = *reinterpret_cast<const float4*>(slot.v + (size_t)h * slot.cap * HD + r);
        st4_bf16(kb + (size_t)h * L * HD + r, kx);
        st4_bf16(vb + (size_t)h * L * HD + r, vx);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
cudaError_t launch_gqa_prefill(dz_ctx* ctx, int layer, int seq, int64_t T, int64_t rope_pos0, const uint16_t* q_gate,
                               const uint16_t* k, const uint16_t* v, const float* q_gate_f, const float* k_f,
                               const float* v_f, float* out, cudaStream_t st, int* n_launch) {
    const LayerState& Lr = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
    const int64_t base = Lr.len[seq];
    const int64_t L = base + T;
    const KvSlot slot = Lr.h_kv[seq];
    const size_t qb_elems = (size_t)nq * T * HD, kb_elems = (size_t)kvc * L * HD;
    cudaError_t e = ensure_prefill_scratch(ctx, (qb_elems + 2 * kb_elems) * 2 + 4096);
    if (e != cudaSuccess) return e;
    __nv_bfloat16* qb = static_cast<__nv_bfloat16*>(ctx->pf);
    __nv_bfloat16* kb = qb + qb_elems;
    __nv_bfloat16* vb = kb + kb_elems;
    const bool bf = q_gate != nullptr;
    if (bf)
        pf_prep_kernel<__nv_bfloat16><<<(unsigned)T, 256, 0, st>>>(
            kvc, T, base, rope_pos0, slot, Lr.q_norm, Lr.k_norm, ctx->rope, reinterpret_cast<const __nv_bfloat16*>(q_gate),
            reinterpret_cast<const __nv_bfloat16*>(k), reinterpret_cast<const __nv_bfloat16*>(v), qb, kb, vb, L,
            ctx->cfg.rms_eps);
    else
        pf_prep_kernel<float><<<(unsigned)T, 256, 0, st>>>(kvc, T, base, rope_pos0, slot, Lr.q_norm, Lr.k_norm, ctx->rope,
                                                          q_gate_f, k_f, v_f, qb, kb, vb, L, ctx->cfg.rms_eps);
    *n_launch += 1;
    if (base > 0) {
        pf_prior_kernel<<<ctx->n_sm * 4, 256, 0, st>>>(kvc, base, slot, kb, vb, L);
        *n_launch += 1;
    }
    CUtensorMap mq, mk, mv;
    if (!pf::make_map<__nv_bfloat16>(&mq, qb, T, nq, pf::BM) || !pf::make_map<__nv_bfloat16>(&mk, kb, L, kvc, pf::BN) ||
        !pf::make_map<__nv_bfloat16>(&mv, vb, L, kvc, 32))
        return cudaErrorInvalidValue;
    const int n_qt = (int)((T + pf::BM - 1) / pf::BM);
    const int sc = ctx->cfg.qtile_split_count, si = ctx->cfg.qtile_split_index;
    const int n_own = n_qt > si ? (n_qt - 1 - si) / sc + 1 : 0;
    const size_t smem = sizeof(pf::Smem) + 1024;
    const pf::OneSequence map{T, base, si, sc};
    using B = __nv_bfloat16;
    if (bf) {
        auto kernel = pf_attn_kernel<B, float, B, pf::OneSequence>;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (n_own > 0)
            kernel<<<n_own * nq, pf::NTHREADS, smem, st>>>(mq, mk, mv, map, kvc, reinterpret_cast<const B*>(q_gate), out,
                                                           ctx->d_err);
    } else {
        auto kernel = pf_attn_kernel<float, float, B, pf::OneSequence>;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (n_own > 0)
            kernel<<<n_own * nq, pf::NTHREADS, smem, st>>>(mq, mk, mv, map, kvc, q_gate_f, out, ctx->d_err);
    }
    *n_launch += 1;
    return cudaGetLastError();
}

}  // namespace dz
