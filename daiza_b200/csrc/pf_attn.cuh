// pf_attn.cuh -- causal flash attention on tcgen05 for prompts: the kernel behind
// gqa_prefill.cu (f32 caches: bf16 operands, one sequence) and q4_prefill.cu (4-bit
// caches: f16 operands, packed sequences).  E is the operand type, Map names each CTA's
// query tile (pf::Tile).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "dz_internal.h"
#include "tc_common.cuh"

namespace dz {

namespace pf {

constexpr int BM = 128;        // query rows per CTA
constexpr int BN = 128;        // keys per block (S = Q K^T runs as M128 x N128 products)
constexpr int NK = 5;          // K ring: slots of one 64-dim box of a key block (128 x 64 bf16, 16 KB)
constexpr int NV = 4;          // V ring: slots of 32 keys x 256 dims (4 boxes of 32 x 64 bf16, 16 KB)
constexpr int NTHREADS = 352;  // warps 0-7 softmax, warp 8 TMA of Q and K, warp 9 MMA, warp 10 TMA of V
// TMEM columns: S buffers [0,128) and [128,256) (f32); P of a block (bf16 pairs)
// overwrites the first 64 columns of its own S buffer; O accumulator [256,512)
__host__ __device__ constexpr uint32_t S_COL(int st) { return 128u * (uint32_t)st; }
constexpr uint32_t O_COL = 256;
constexpr float RESCALE_THRESHOLD = 8.0f;   // log2 units

struct alignas(1024) Smem {
    uint16_t q[4][BM][64];               // 4 boxes of 64 dims, 16 KB each (bf16 or f16)
    uint16_t k[NK][BN][64];              // K ring
    uint16_t v[NV][4][32][64];           // V ring
    uint64_t q_full;
    uint64_t k_full[NK], k_empty[NK], v_full[NV], v_empty[NV];
    uint64_t s_full[2], p_full[2], pv_done[2];
    float red_max[2][2][BM];             // [block parity][column half][row] partial row maxima
    float red_l[2][BM];                  // [column half][row] partial row sums
    uint32_t tmem_base;
};
static_assert(offsetof(Smem, k) % 1024 == 0 && offsetof(Smem, v) % 1024 == 0, "swizzle atoms need 1 KB alignment");

using namespace tc;

// Instruction descriptor, kind::f16: A and B of the operand type, f32 accumulator.
template <typename E>
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool b_mn_major) {
    const uint32_t type = std::is_same<E, __half>::value ? 0u : 1u;   // f16 0, bf16 1
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// three-input maximum (sm_100)
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// packed f32x2 arithmetic on register pairs (sm_100)
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_split(uint64_t r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t sub_f2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);   // .x = a (low half)
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);   // .x = a (low half)
    return *reinterpret_cast<const uint32_t*>(&v);
}

// One query tile of a CTA: rows [q0, q0 + 128) of a sequence of T new tokens behind `base`
// keys.  row: the tile's first row in the Q map, q_gate and out; key: the sequence's first
// row in the K and V maps.
struct Tile { int64_t q0, T, base, row, key; };
// One sequence.  Heaviest (latest) query tiles first; with a split, a context owns the
// tiles qt % split_cnt == split_idx (interleaved: balanced causal work).
struct OneSequence {
    int64_t T, base;
    int split_idx, split_cnt;
    __device__ __forceinline__ Tile tile(int i) const {
        const int n_qt = (int)((T + BM - 1) / BM);
        const int last_own = (n_qt - 1) - (((n_qt - 1) % split_cnt) - split_idx + split_cnt) % split_cnt;
        const int64_t q0 = (int64_t)(last_own - split_cnt * i) * BM;
        return {q0, T, base, q0, 0};
    }
};

}  // namespace pf

template <typename Tin>
__device__ __forceinline__ float4 ld4(const Tin* p);
template <>
__device__ __forceinline__ float4 ld4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 ld4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&u.x);
    const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&u.y);
    return make_float4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
}
__device__ __forceinline__ void st4_bf16(__nv_bfloat16* p, float4 x) {
    uint2 u;
    u.x = pf::pack_bf16(x.x, x.y);
    u.y = pf::pack_bf16(x.z, x.w);
    *reinterpret_cast<uint2*>(p) = u;
}

__device__ __forceinline__ void st4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void st4(__nv_bfloat16* p, float4 x) { st4_bf16(p, x); }

// ---------------------------------------------------------------------------
// attention: one CTA per (q head, 128-row query tile); see gqa_prefill.cu for its parts
// ---------------------------------------------------------------------------
template <typename Tg, typename To, typename E, typename Map>
__global__ void __launch_bounds__(pf::NTHREADS, 1) pf_attn_kernel(const __grid_constant__ CUtensorMap tm_q,
                                                                   const __grid_constant__ CUtensorMap tm_k,
                                                                   const __grid_constant__ CUtensorMap tm_v,
                                                                   const __grid_constant__ Map map, int kvc,
                                                                   const Tg* __restrict__ q_gate,
                                                                   To* __restrict__ out, int* err) {
    using namespace pf;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // dynamic smem is only guaranteed 16-byte aligned: round up to 1 KB
    // offset the shared-memory pointer itself (integer arithmetic on the address
    // would turn every later access into a generic one)
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nq = GRP * kvc;
    const Tile tl = map.tile((int)(blockIdx.x / nq));
    const int qh = (int)(blockIdx.x % nq);
    const int kvh = qh / GRP;
    const int64_t q0 = tl.q0, T = tl.T, base = tl.base;
    const int64_t q_last = std::min<int64_t>(q0 + BM, T) - 1;         // last valid query row (token index)
    const int nblk = (int)((base + q_last) / BN) + 1;                  // key blocks touching the causal range

    if (warp == 0) {
        tmem_alloc(&sm.tmem_base, 512);
    }
    if (tid == 0) {
        mbar_init(&sm.q_full, 1);
        for (int i = 0; i < NK; ++i) {
            mbar_init(&sm.k_full[i], 1);
            mbar_init(&sm.k_empty[i], 1);
        }
        for (int i = 0; i < NV; ++i) {
            mbar_init(&sm.v_full[i], 1);
            mbar_init(&sm.v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 2 * BM);
            mbar_init(&sm.pv_done[i], 1);
        }
        fence_mbar_init();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    bool ok = true;

    if (warp == 8) {
        // ---------------- TMA producer of Q and K boxes ----------------
        if (lane == 0) {
            mbar_arrive_expect_tx(&sm.q_full, BM * HD * 2);
            for (int b = 0; b < 4; ++b) tma_load_3d(&sm.q[b][0][0], &tm_q, 64 * b, (int)tl.row, qh, &sm.q_full);
            for (int idx = 0; idx < 4 * nblk && ok; ++idx) {
                const int slot = idx % NK, j = idx >> 2, b = idx & 3;
                if (idx >= NK && !wait_or_flag(&sm.k_empty[slot], ((idx / NK) - 1) & 1, err, ok)) break;
                mbar_arrive_expect_tx(&sm.k_full[slot], BN * 64 * 2);
                tma_load_3d(&sm.k[slot][0][0], &tm_k, 64 * b, (int)tl.key + j * BN, kvh, &sm.k_full[slot]);
            }
        }
    } else if (warp == 10) {
        // ---------------- TMA producer of V slots: a warp of its own, since a lane that waits for
        // K's slots would hold back the V loads of another lane of its warp ----------------
        if (lane == 0) {
            for (int idx = 0; idx < 4 * nblk && ok; ++idx) {
                const int slot = idx % NV, j = idx >> 2, kg = idx & 3;
                if (idx >= NV && !wait_or_flag(&sm.v_empty[slot], ((idx / NV) - 1) & 1, err, ok)) break;
                mbar_arrive_expect_tx(&sm.v_full[slot], 32 * HD * 2);
                for (int d = 0; d < 4; ++d)
                    tma_load_3d(&sm.v[slot][d][0][0], &tm_v, 64 * d, (int)tl.key + j * BN + 32 * kg, kvh, &sm.v_full[slot]);
            }
        }
    } else if (warp == 9) {
        // ---------------- MMA issuer (one thread) ----------------
        if (lane == 0) {
            constexpr uint32_t ID_QK = idesc<E>(BM, BN, false);
            constexpr uint32_t ID_PV = idesc<E>(BM, HD, true);
            const uint32_t q_s = smem_u32(&sm.q[0][0][0]);
            const uint32_t k_s = smem_u32(&sm.k[0][0][0]);
            const uint32_t v_s = smem_u32(&sm.v[0][0][0][0]);
            auto issue_s = [&](int j) {
                const int st = j & 1;
                for (int b = 0; b < 4; ++b) {
                    const int idx = 4 * j + b, slot = idx % NK;
                    if (!wait_or_flag(&sm.k_full[slot], (idx / NK) & 1, err, ok)) return;
                    fence_after_sync();
#pragma unroll
                    for (int s4 = 0; s4 < 4; ++s4) {
                        const uint32_t off_q = (uint32_t)b * (BM * 128) + (uint32_t)s4 * 32;
                        const uint32_t off_k = (uint32_t)slot * (BN * 128) + (uint32_t)s4 * 32;
                        umma_ss(tmem + S_COL(st), sw128_desc(q_s + off_q, 16, 1024),
                                sw128_desc(k_s + off_k, 16, 1024), ID_QK, (b > 0 || s4 > 0) ? 1u : 0u);
                    }
                    umma_commit(&sm.k_empty[slot]);
                }
                umma_commit(&sm.s_full[st]);
            };
            if (wait_or_flag(&sm.q_full, 0, err, ok)) {
                issue_s(0);
                if (nblk > 1) issue_s(1);
                for (int j = 0; j < nblk && ok; ++j) {
                    const int st = j & 1;
                    if (!wait_or_flag(&sm.p_full[st], (j >> 1) & 1, err, ok)) break;
                    for (int kg = 0; kg < 4 && ok; ++kg) {
                        const int idx = 4 * j + kg, slot = idx % NV;
                        if (!wait_or_flag(&sm.v_full[slot], (idx / NV) & 1, err, ok)) break;
                        fence_after_sync();
#pragma unroll
                        for (int s2 = 0; s2 < 2; ++s2) {
                            // B = V[16 keys][256 dims], MN-major: 64-dim boxes 4 KB apart (LBO),
                            // 8-key swizzle atoms 1 KB apart (SBO); A = P columns of those keys
                            umma_ts(tmem + O_COL, tmem + S_COL(st) + 8 * (2 * kg + s2),
                                    sw128_desc(v_s + (uint32_t)slot * (32 * HD * 2) + (uint32_t)s2 * 16 * 128,
                                               32 * 128, 1024),
                                    ID_PV, (j > 0 || kg > 0 || s2 > 0) ? 1u : 0u);
                        }
                        umma_commit(&sm.v_empty[slot]);
                    }
                    umma_commit(&sm.pv_done[st]);
                    if (j + 2 < nblk) issue_s(j + 2);
                }
            }
        }
    } else {
        // ---------------- softmax: 8 warps, thread = (query row, key half) ----------------
        const int r = 32 * (warp & 3) + lane;               // TMEM lane = query row
        const int hf = warp >> 2;                           // keys [64 hf, 64 hf + 64) of a block
        const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
        const int64_t qpos = base + q0 + r;                 // absolute position of this query row
        float m_run = -INFINITY, l_run = 0.0f;              // m identical in both halves; l partial per half
        for (int j = 0; j < nblk; ++j) {
            const int st = j & 1;
            if (!wait_or_flag(&sm.s_full[st], (j >> 1) & 1, err, ok)) break;
            fence_after_sync();
            float s[64];
            {
                uint32_t raw[64];
                tmem_ld32_async(tmem + lane_off + S_COL(st) + 64 * hf, raw);
                tmem_ld32_async(tmem + lane_off + S_COL(st) + 64 * hf + 32, raw + 32);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = __uint_as_float(raw[c]);
            }
            // causal mask: keys k0 + c with c > lim are in the future (only blocks on the diagonal)
            const int64_t lim64 = qpos - ((int64_t)j * BN + 64 * hf);
            if (lim64 < 63) {
                const int lim = lim64 < -1 ? -1 : (int)lim64;
#pragma unroll
                for (int c = 0; c < 64; ++c) s[c] = c > lim ? -INFINITY : s[c];
            }
            float mx;
            {
                float a0 = s[0], a1 = s[1], a2 = s[2], a3 = s[3];
#pragma unroll
                for (int c = 4; c < 64; c += 8) {
                    a0 = max3f(a0, s[c], s[c + 1]);
                    a1 = max3f(a1, s[c + 2], s[c + 3]);
                    a2 = max3f(a2, s[c + 4], s[c + 5]);
                    a3 = max3f(a3, s[c + 6], s[c + 7]);
                }
                mx = fmaxf(max3f(a0, a1, a2), a3);
            }
            sm.red_max[st][hf][r] = mx;
            named_bar_sync(1, 256);                          // also: every S read of this block is done
            mx = fmaxf(mx, sm.red_max[st][hf ^ 1][r]);
            const float m_new = fmaxf(m_run, mx);
            if (m_new > m_run + RESCALE_THRESHOLD) {
                // lazy rescale: the running max moved a lot -- scale l and this half-row of O
                const float f = ex2(m_run - m_new);
                l_run *= f;
                if (j > 0) {
                    const int pj = (j - 1) & 1;
                    if (!wait_or_flag(&sm.pv_done[pj], ((j - 1) >> 1) & 1, err, ok)) break;
                    fence_after_sync();
#pragma unroll 1
                    for (int c = 128 * hf; c < 128 * hf + 128; c += 32) {
                        float o[32];
                        uint32_t ob[32];
                        tmem_ld32(tmem + lane_off + O_COL + c, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) ob[i] = __float_as_uint(o[i] * f);
                        tmem_st32(tmem + lane_off + O_COL + c, ob);
                    }
                }
                m_run = m_new;
            }
            uint32_t pk[32];
            {
                const uint64_t mm = f2(m_run, m_run);
                uint64_t acc0 = f2(0.0f, 0.0f), acc1 = acc0;
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    float x0, x1, x2, x3;
                    f2_split(sub_f2(f2(s[c], s[c + 1]), mm), x0, x1);
                    f2_split(sub_f2(f2(s[c + 2], s[c + 3]), mm), x2, x3);
                    const float p0 = ex2(x0), p1 = ex2(x1), p2 = ex2(x2), p3 = ex2(x3);
                    acc0 = add_f2(acc0, f2(p0, p1));
                    acc1 = add_f2(acc1, f2(p2, p3));
                    pk[c / 2] = pack2<E>(p0, p1);
                    pk[c / 2 + 1] = pack2<E>(p2, p3);
                }
                float u0, u1;
                f2_split(add_f2(acc0, acc1), u0, u1);
                l_run += u0 + u1;
            }
            // P of this block goes over the first 64 columns of its own S buffer (the
            // previous reader of these columns, PV(j-2), completed before S(j) did)
            tmem_st32(tmem + lane_off + S_COL(st) + 32 * hf, pk);
            fence_before_sync();
            mbar_arrive(&sm.p_full[st]);
        }
        // epilogue: O / l * sigmoid(gate); this thread covers dims [128 hf, 128 hf + 128)
        sm.red_l[hf][r] = l_run;
        named_bar_sync(1, 256);
        const float l_tot = l_run + sm.red_l[hf ^ 1][r];
        if (ok) {
            const int jl = nblk - 1;
            if (wait_or_flag(&sm.pv_done[jl & 1], (jl >> 1) & 1, err, ok)) {
                fence_after_sync();
                const int64_t t = tl.row + r;
                const float inv_l = 1.0f / l_tot;
#pragma unroll 1
                for (int c = 128 * hf; c < 128 * hf + 128; c += 32) {
                    float o[32];
                    tmem_ld32(tmem + lane_off + O_COL + c, o);
                    if (q0 + r < T) {
                        const Tg* g = q_gate + (t * nq + qh) * QG_ROW + HD + c;
                        To* dst = out + (t * nq + qh) * HD + c;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 gv = ld4<Tg>(g + i);
                            float4 y;
                            y.x = o[i + 0] * inv_l * sigmoidf_acc(gv.x);
                            y.y = o[i + 1] * inv_l * sigmoidf_acc(gv.y);
                            y.z = o[i + 2] * inv_l * sigmoidf_acc(gv.z);
                            y.w = o[i + 3] * inv_l * sigmoidf_acc(gv.w);
                            st4(dst + i, y);
                        }
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

namespace pf {
// bf16 or f16 tensor [d2][d1][256] with a (64 x rows x 1) box, 128-byte swizzle
template <typename E>
bool make_map(CUtensorMap* m, const void* base, int64_t d1, int64_t d2, int box_rows) {
    EncodeTiledFn fn = tensor_map_encoder();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)d1, (cuuint64_t)d2};
    cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)d1 * HD * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, std::is_same<E, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
}  // namespace pf

}  // namespace dz
