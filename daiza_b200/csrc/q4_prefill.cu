// q4_prefill.cu -- prompts into 4-bit KV caches: packed sequences of different lengths,
// rotary positions of three axes, causal attention over the held rows.
//
// Reference: Daiza-engine/src/model/forward.rs:599-721 (parallel GQA prefill), for several
// sequences at once.  Token t of a sequence with `base` cached rows attends over rows
// 0 .. base + t as the cache holds them (4 bits), its own row included: the same as one
// decode call per token.
//
// Two kernels:
//   1. q4_pf_prep : Q normed, rotated, scaled (by a power of two, too, that keeps it inside f16
//                   whatever the norm weights: q_up), as f16 [head][token][256]; K (normed, rotated,
//                   f64) and V quantised into the sequences' tiles; and every held row, old
//                   and new, as f16 [kv head][key][256] -- exact -- each sequence padded with
//                   zeros to whole blocks of 128 keys, so that a block never meets another
//                   sequence's values.  Blocks of three kinds, all independent.
//   2. q4_pf_attn : causal flash attention on tcgen05, f16 operands (K and V are exact, Q and P
//                   rounded to 11 bits; bf16's 8 would cost the output's last bits), two
//                   heads of a group to a CTA pair.
#include <cuda.h>
#include <algorithm>
#include <cstddef>

#include "q4.cuh"
#include "tc_common.cuh"

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

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);   // a in the low half
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void load_row(const T* p, float (&x)[8]) {
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

// 8192 bf16 tokens: 77 us for 0.28 GB (3.6 TB/s).  Bound by issue (59 % of the slots, at two
// blocks per SM; more blocks spill): norms, rotation, the codes and their f16 values.
constexpr int PREP_WARPS = 16, PREP_ROWS = 4;    // query rows that a warp has in flight

// Blocks [0, at0 kvc / key_heads): a tile of new rows and key_heads kv heads, a warp per position.
// Then (old0 kvc) blocks: a tile of cached rows or padding, a warp per position.
// Then: a warp per token and q_heads of its heads.
template <typename T>
__global__ void __launch_bounds__(32 * PREP_WARPS, 2)
    q4_pf_prep_kernel(const __grid_constant__ Prompt d, const __grid_constant__ RopeAxes axes, int kvc,
                      const Q4Slot* __restrict__ slots, const int32_t* __restrict__ pos, const float* __restrict__ q_norm,
                      const float* __restrict__ k_norm, const T* __restrict__ q_gate, const T* __restrict__ k,
                      const T* __restrict__ v, __half* __restrict__ qf, __half* __restrict__ kf, __half* __restrict__ vf,
                      int key_heads, int q_heads, bool track, float eps, float q_up) {
    __shared__ TileMerge merge;
    __shared__ double2 cs[PREP_WARPS][ROPE / 2];
    __shared__ float2 csf[PREP_WARPS][ROPE / 2];
    // the attention grid's CTAs may take their places as these blocks leave
    asm volatile("griddepcontrol.launch_dependents;");
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
    const int shares = kvc / key_heads;
    if (block < (int64_t)d.at0[d.n] * shares) {
        const int at = (int)(block / shares), kvh0 = (int)(block - (int64_t)at * shares) * key_heads;
        const int s = last_at_or_before(d.at0, d.n, at);
        const int base = d.base[s], t16 = (base >> 4) + (at - d.at0[s]), slot_pos = t16 * Q4_TILE + warp;
        const Q4Slot slot = slots[d.sid[s]];
        const bool mine = slot_pos >= base && slot_pos < base + d.T(s);
        const int64_t row = d.row0[s] + (slot_pos - base);
        int p[3];
        merge.begin();
        if (mine) {
            angles_at(s, row, p);
            csf[warp][lane] = rope_cs_f32(axes, lane, p[0], p[1], p[2]);
        }
#pragma unroll 1
        for (int kvh = kvh0; kvh < kvh0 + key_heads; ++kvh) {
            uint8_t* tile = slot.tile(kvh, t16);
            __syncthreads();
            if (mine) {
                float x[8], y[8];
                load_row(k + (row * kvc + kvh) * HD + 8 * lane, x);
                load_row(v + (row * kvc + kvh) * HD + 8 * lane, y);
                const size_t out = ((size_t)kvh * keys + d.key0[s] + slot_pos) * HD + 8 * lane;
                uint32_t code[8];
                uint32_t sb = quantise_key(x, k_norm, csf[warp], cs[warp], axes, p[0], p[1], p[2], eps, lane, code);
                put_k(tile, warp, lane, code, sb);
                *reinterpret_cast<uint4*>(kf + out) = held(code, sb);
                sb = quantise(y, code);
                merge.add(warp, lane, code);
                put_v_scale(tile, warp, lane, sb);
                *reinterpret_cast<uint4*>(vf + out) = held(code, sb);
                if (track && lane == 0) slot.wts[(size_t)kvh * slot.cap + slot_pos] = 0.0f;
            }
            merge.end(tile, base - t16 * Q4_TILE, base + d.T(s) - t16 * Q4_TILE);
        }
        return;
    }
    block -= (int64_t)d.at0[d.n] * shares;
    if (block < (int64_t)d.old0[d.n] * kvc) {
        const int ot = (int)(block / kvc), kvh = (int)(block - (int64_t)ot * kvc);
        const int s = last_at_or_before(d.old0, d.n, ot);
        const int i = ot - d.old0[s], cached = d.cached_tiles(s);
        const int t16 = i < cached ? i : d.first_pad_tile(s) + (i - cached), at = t16 * Q4_TILE + warp;
        const bool old = i < cached;
        if (old ? at >= d.base[s] : at < d.base[s] + d.T(s)) return;   // a new row
        // (in the last cached tile, words that hold old and new rows may be written meanwhile by
        // the block that appends: the old rows' bits stay the same)
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
    const int parts = (nq + q_heads - 1) / q_heads;
    const int64_t task = block * PREP_WARPS + warp, row = task / parts;
    if (row >= tokens) return;
    const int h_first = (int)(task - row * parts) * q_heads, h1 = min(nq, h_first + q_heads);
    int p[3];
    angles_at(pos ? 0 : last_at_or_before(d.row0, d.n, (int)row), row, p);
    float2 c4[4];
    spread_pairs(rope_cs_f32(axes, lane, p[0], p[1], p[2]), c4, lane);
    float w[8];
    load_split(q_norm, lane, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] *= 0.0625f * LOG2E * q_up;   // scores in log2 units, times q_up
    auto store_q = [&](int h, const float (&x)[8]) {
        __half* out = qf + ((size_t)h * tokens + row) * HD;
        *reinterpret_cast<uint2*>(out + split_dim(lane, 0)) = make_uint2(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]));
        *reinterpret_cast<uint2*>(out + split_dim(lane, 1)) = make_uint2(pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
    };
    uint32_t far = 0;                            // heads whose row is out of range
#pragma unroll 1
    for (int h0 = h_first; h0 < h1; h0 += PREP_ROWS) {
        SplitRow<T> in[PREP_ROWS];
#pragma unroll
        for (int i = 0; i < PREP_ROWS; ++i)
            if (h0 + i < h1) in[i].load(q_gate + (row * nq + h0 + i) * QG_ROW, lane);
#pragma unroll
        for (int i = 0; i < PREP_ROWS; ++i) {
            if (h0 + i >= h1) break;
            float x[8];
            in[i].values(x);
            if (!norm_rotate_split(x, w, c4, eps, lane)) far |= 1u << (h0 + i);
            store_q(h0 + i, x);
        }
    }
    for (; far; far &= far - 1) {
        const int h = __ffs(far) - 1;
        float x[8];
        load_split(q_gate + (row * nq + h) * QG_ROW, lane, x);
        norm_rotate_far(x, w, c4, eps, lane);
        store_q(h, x);
    }
}

// ---------------------------------------------------------------------------
// Attention.  A cluster of two CTAs takes a query tile of 128 tokens of two q heads of one
// group, a head each, with tcgen05.mma.cta_group::2: M = 256 rows, each CTA's 128 in its own
// TMEM, and every K and V block fetched once for both, half by each CTA.  (One CTA per
// tile had to take in 128 KB per block of 128 keys, about 2000 cycles at an SM's 64
// bytes a cycle, beside 2100 cycles of products: 3300 cycles a block.)
//   warps 0-7  softmax: thread = (query row, half of a block's 128 keys); scores in log2
//              units, running max rescaled lazily (only when it grows by more than 8), P as f16
//              over its S columns, finally O / l to the output warps
//   warp 8     TMA of Q and of this CTA's 64 keys of each K block (slots of 64 dims)
//   warp 9     (first CTA) issues S = Q K^T (N = 128, K = 256) into one of two TMEM buffers
//              and O += P V (N = 256, K = 128, P from TMEM)
//   warp 10    TMA of this CTA's 128 dims of each V block (slots of 32 keys)
//   warps 12-15  outputs: O / l from shared memory, times the gate's sigmoid, in whole rows.  bf16
//              outputs pass as f16 (2^-11, an eighth of what bf16 rounds; times 8, which keeps |V| <=
//              7 * 896 in range and small values' bits), f32 ones as f32, one half of the dims
//              after the other
// A cluster takes several query tiles in turn; while the outputs of one leave, the next one's
// queries are fetched and its first blocks worked on.  (A cluster per tile, the softmax warps
// writing the outputs: packed prompts of 1-1500 took 378 us, all of the call, instead of 240:
// set-up and outputs were 15 us of each tile's time, next to 1.3 us per block of keys.)
// Bound by the products and the softmax together: a block of 128 keys takes 2270 cycles, of
// which the products 2048; the softmax of one block (1950 cycles, 1100 of them exponentials)
// runs beside the products of another.  8192 tokens: 825 GFLOP, 1.35-1.5 PFLOP/s with the SM
// clock at 1.6-1.8 GHz.
// The first CTA's barriers count both CTAs' bytes and arrivals; the products' completion
// goes to both.  Every wait is bounded; a CTA that gave one up still meets its barriers.
// ---------------------------------------------------------------------------
namespace attn {
using namespace tc;

constexpr int BM = 128, BN = 128;                // query rows of a CTA, keys of a block
constexpr int NK = 6, NV = 5;                    // ring slots of 8 KB (a block is 4 of each)
constexpr int NTHREADS = 512;
__host__ __device__ constexpr uint32_t S_COL(int st) { return 128u * (uint32_t)st; }
constexpr uint32_t O_COL = 256;
constexpr float OUT_SCALE = 8.0f;
// The matrix instruction adds to its f32 accumulator with truncation: 2e-7 of the sum an instruction of 16 keys, all one
// way (131072 keys of like values came out 8.4e-4 short).  So O starts anew every STRETCH blocks of keys, and what it
// held is added up, rounded to nearest, in memory: 5e-5 short at any length, a fifth of what P's rounding does.  1024
// tokens behind 65000 take 1470 us so, 1405 without (1450 with 128 blocks).  A launch without a sequence that long (LONG =
// false) has none of it in its code: packed prompts of 1-1500 took 248.7 us with it, 243.2 without.
constexpr int STRETCH = 64;
constexpr int64_t PART_BYTES = (int64_t)BM * HD * sizeof(float);   // a CTA's sums, [dim][row]
// log2 units.  P is taken times 2^P_LOG2 against a maximum that may be stale by RESCALE_THRESHOLD: at most 2^15, inside f16,
// and keys 31 units below the maximum still count (without it those below 25 were 0 in P, but not in its sum: 200000 of
// them, 0.4 % of the weight, were lost).
constexpr float RESCALE_THRESHOLD = 8.0f, P_LOG2 = 7.0f;

struct alignas(1024) Smem {
    uint16_t q[4][BM][64];                       // 4 boxes of 64 dims, 16 KB each
    uint16_t k[NK][BN / 2][64];
    uint16_t v[NV][2][32][64];
    uint4 out[BM][32];                           // O / l, a row's 16-byte words swizzled: 256 dims as f16, or 128 as f32
    uint64_t q_full, q_empty, out_full[2], out_empty[2];   // out: of either half of the dims (f32), [0] of both (bf16)
    uint64_t k_full[NK], k_empty[NK], v_full[NV], v_empty[NV];
    uint64_t s_full[2], p_full[2], pv_done[2];
    float red_max[2][2][BM];                     // [block parity][key half][row] partial row maxima
    float red_l[2][BM];                          // [key half][row] partial row sums
    uint32_t tmem_base;
};
constexpr int SMEM_BYTES = (int)sizeof(Smem) + 1024;           // the kernel rounds its address up to 1 KB
static_assert(offsetof(Smem, k) % 1024 == 0 && offsetof(Smem, v) % 1024 == 0, "swizzle atoms need 1 KB alignment");

// ---- the pair's forms of the PTX wrappers ------------------------------------------
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// a load into this CTA, counted on a barrier of the pair (a shared::cluster address)
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void alloc(uint32_t* dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// Issued by the one lane whose `go` is set, in code that its whole warp runs: the operands
// then stay in uniform registers (issued under `if (lane == 0)` an instruction took about
// 100 cycles, more than the product itself).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t go;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(go));
    return go;
}
// the issued products' completion, to this barrier of both CTAs
__device__ __forceinline__ void commit(uint32_t go, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\tsetp.ne.b32 q, %1, 0;\n\tmov.b16 m, 3;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
        ::"r"(bar), "r"(go) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t go, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t go, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(go) : "memory");
}
// f16 A and B, f32 accumulator; B optionally MN-major
constexpr uint32_t idesc(int M, int N, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// What crosses CTAs under these barriers is TMEM and TMA data, ordered by tcgen05 fences and
// by the copies' own completion: a release or acquire at cluster scope would only add
// memory barriers (they cost a tenth of the kernel).
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, bool& ok) {
    return wait_or_flag(bar, parity, err, ok);
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x without the special-function unit, x at most 15: x = n + f with n nearest, a polynomial of
// degree 4 for 2^f (least squares weighted towards the smallest largest error: 2.6e-6, far below P's
// f16 rounding), n added to its exponent.  Below -126: 2^-126.  A quarter of the exponentials
// this way: packed prompts of 1-1500 take 244.2 us (246.8 without), 2000 tokens after 5555 248.2 (250.4), 1024 behind
// 65000 1480 (1492); two runs of one differ by 0.2 %.
__device__ __forceinline__ void ex2_poly(uint64_t x, float& p0, float& p1) {
    float a, b;
    unpack2(x, a, b);
    x = pack2(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    const uint64_t big = pack2(12582912.0f, 12582912.0f);                 // 1.5 * 2^23: sums are rounded to integers
    const uint64_t t = add2(x, big), f = sub2(x, sub2(t, big));
    uint64_t y = fma2(pack2(0.0095701f, 0.0095701f), f, pack2(0.05591786f, 0.05591786f));
    y = fma2(y, f, pack2(0.24024745f, 0.24024745f));
    y = fma2(y, f, pack2(0.69312181f, 0.69312181f));
    y = fma2(y, f, pack2(0.99999926f, 0.99999926f));
    float t0, t1;
    unpack2(t, t0, t1);
    unpack2(y, a, b);
    p0 = __uint_as_float(__float_as_uint(a) + (__float_as_uint(t0) << 23));
    p1 = __uint_as_float(__float_as_uint(b) + (__float_as_uint(t1) << 23));
}
// (a sigmoid(x), b sigmoid(y)) / OUT_SCALE of f16 a and b, to 2^-20 or so, below the products' f16 rounding: 1 / (8 + 2^(3 - x
// log2 e)).  (One reciprocal of both denominators' product has to be kept from overflowing: it took as long.)
__device__ __forceinline__ float2 gate2(uint32_t ab, float x, float y) {
    static_assert(OUT_SCALE == 8.0f, "the exponent's 3");
    float s, t, u, w, g, h;
    unpack2(fma2(pack2(x, y), pack2(-LOG2E, -LOG2E), pack2(3.0f, 3.0f)), s, t);
    unpack2(add2(pack2(ex2(s), ex2(t)), pack2(OUT_SCALE, OUT_SCALE)), u, w);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g) : "f"(u));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(w));
    const float2 o = __half22float2(*reinterpret_cast<const __half2*>(&ab));
    float2 out;
    unpack2(mul2(pack2(o.x, o.y), pack2(g, h)), out.x, out.y);
    return out;
}
// four f32 values times the gates' sigmoids
__device__ __forceinline__ float4 gate4(uint4 o, float4 x) {
    const float v[4] = {__uint_as_float(o.x), __uint_as_float(o.y), __uint_as_float(o.z), __uint_as_float(o.w)};
    const float g[4] = {x.x, x.y, x.z, x.w};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(-LOG2E * g[i])));
        y[i] = v[i] * r;
    }
    return make_float4(y[0], y[1], y[2], y[3]);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, float4 a, float4 b) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
}

// One query tile: rows [q0, q0 + 128) of a sequence of T new tokens behind `base` keys.  row:
// the tile's first row in the Q map, q_gate and out; key: the sequence's first row in K and V.
struct Tile { int64_t q0, T, base, row, key; };
// Packed sequences, those with the most keys first and their latest query tiles first: the
// heaviest tiles start first.  A context owns the tiles t % split_cnt == split_idx.
struct Packed {
    int n, split_idx, split_cnt;
    int32_t first[MAXB + 1];                     // query tiles before the i-th sequence of this order
    int32_t T[MAXB], base[MAXB], row[MAXB], key[MAXB];
    static int own_tiles(int64_t T, int idx, int cnt) {
        const int n_qt = (int)((T + BM - 1) / BM);
        return n_qt > idx ? (n_qt - 1 - idx) / cnt + 1 : 0;
    }
    __device__ __forceinline__ Tile tile(int i) const {
        const int s = last_at_or_before(first, n, i);
        const int own = first[s + 1] - first[s];
        const int64_t q0 = (int64_t)(split_idx + split_cnt * (own - 1 - (i - first[s]))) * BM;
        return {q0, T[s], base[s], row[s] + q0, key[s]};
    }
};

template <typename T, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NTHREADS, 1)
    q4_pf_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Packed map, int kvc,
                      const T* __restrict__ q_gate, T* __restrict__ out, float* __restrict__ part, float q_down, int* err) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // dynamic shared memory is only 16-byte aligned: round up to 1 KB (the same place in both CTAs)
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    // registers by warpgroup (with 56 / 104 / 176 the f32 kernel spills: packed prompts took 218 us instead of 183)
    constexpr int REGS_LOAD = sizeof(T) == 4 ? 72 : 56, REGS_OUT = 104, REGS_SOFTMAX = sizeof(T) == 4 ? 168 : 176;
    static_assert(REGS_LOAD + REGS_OUT + 2 * REGS_SOFTMAX <= 65536 / BM, "a warpgroup each of the first two, two of softmax");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nq = GRP * kvc, pairs = nq / 2, rank = blockIdx.x & 1;
    // the cluster's tiles, heaviest first: in rounds over all clusters, there and back
    const int clusters = gridDim.x / 2, cluster = blockIdx.x / 2, total = map.first[map.n] * pairs;
    int round = 0, qh, kvh, nblk;                                      // nblk: key blocks that touch the causal range
    Tile tl;
    auto next_tile = [&]() -> bool {
        const int at = round * clusters + (round & 1 ? clusters - 1 - cluster : cluster);
        if (at >= total) return false;
        tl = map.tile(at / pairs);
        qh = 2 * (at % pairs) + rank;
        kvh = qh / GRP;
        nblk = (int)((tl.base + min(tl.q0 + BM, tl.T) - 1) / BN) + 1;
        ++round;
        return true;
    };

    if (tid == 0) {
        mbar_init(&sm.q_full, 1);
        mbar_init(&sm.q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.out_full[i], sizeof(T) == 4 ? 4 : 8);        // the softmax warps of this CTA (f32: of one half)
            mbar_init(&sm.out_empty[i], 4);                            // the output warps
        }
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
            mbar_init(&sm.p_full[i], 16);                              // the softmax warps of both CTAs
            mbar_init(&sm.pv_done[i], 1);
        }
        fence_mbar_init();
    }
    if (warp == 0) alloc(&sm.tmem_base, 512);
    fence_before_sync();
    __syncthreads();
    cluster_sync();
    fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    bool ok = true;

    if (warp >= 8 && warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_LOAD));
    if (warp == 8) {
        // ---------------- TMA of Q and K ----------------
        if (lane == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");         // for q4_pf_prep
            const uint32_t qb = peer_addr(&sm.q_full, 0);
            int slot = 0;
            uint32_t phase = 1;                                        // of the slot before: passes on a fresh ring
            while (ok && next_tile()) {
                if (round > 1 && !wait(&sm.q_empty, round & 1, err, ok)) break;
                if (rank == 0) mbar_arrive_expect_tx(&sm.q_full, 2 * BM * HD * 2);
                for (int b = 0; b < 4; ++b) tma_load(&sm.q[b][0][0], &tm_q, 64 * b, (int)tl.row, qh, qb);
                for (int idx = 0; idx < 4 * nblk; ++idx) {
                    const int j = idx >> 2, b = idx & 3;
                    if (!wait(&sm.k_empty[slot], phase, err, ok)) break;
                    if (rank == 0) mbar_arrive_expect_tx(&sm.k_full[slot], BN * 64 * 2);
                    tma_load(&sm.k[slot][0][0], &tm_k, 64 * b, (int)tl.key + j * BN + rank * (BN / 2), kvh,
                             peer_addr(&sm.k_full[slot], 0));
                    if (++slot == NK) {
                        slot = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 10) {
        // ---------------- TMA of V ----------------
        if (lane == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int slot = 0;
            uint32_t phase = 1;
            while (ok && next_tile()) {
                for (int idx = 0; idx < 4 * nblk; ++idx) {
                    const int j = idx >> 2, kg = idx & 3;
                    if (!wait(&sm.v_empty[slot], phase, err, ok)) break;
                    if (rank == 0) mbar_arrive_expect_tx(&sm.v_full[slot], 32 * HD * 2);
                    for (int d = 0; d < 2; ++d)
                        tma_load(&sm.v[slot][d][0][0], &tm_v, 128 * rank + 64 * d, (int)tl.key + j * BN + 32 * kg, kvh,
                                 peer_addr(&sm.v_full[slot], 0));
                    if (++slot == NV) {
                        slot = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 9) {
        // ---------------- products (first CTA; the whole warp, one lane issues) ----------------
        if (rank == 0) {
            constexpr uint32_t ID_QK = idesc(2 * BM, BN, false), ID_PV = idesc(2 * BM, HD, true);
            // matrix descriptors count 16 bytes in their low bits: offsets are added
            const uint64_t q_d = sw128_desc(smem_u32(&sm.q[0][0][0]), 16, 1024);
            const uint64_t k_d = sw128_desc(smem_u32(&sm.k[0][0][0]), 16, 1024);
            // V: [16 keys][dims], MN-major: 64-dim boxes 4 KB apart (LBO), 8-key swizzle atoms 1 KB apart (SBO)
            const uint64_t v_d = sw128_desc(smem_u32(&sm.v[0][0][0][0]), 32 * 128, 1024);
            const uint32_t k_empty = smem_u32(&sm.k_empty[0]), v_empty = smem_u32(&sm.v_empty[0]);
            const uint32_t go = elect_one();
            int k_slot = 0, v_slot = 0;
            uint32_t k_phase = 0, v_phase = 0, g = 0;                  // g: blocks of the cluster's earlier tiles
            auto issue_s = [&](int j) {
                const int st = (g + j) & 1;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (!wait(&sm.k_full[k_slot], k_phase, err, ok)) return;
                    fence_after_sync();
                    const uint64_t kd = k_d + (uint64_t)(uint32_t)(k_slot * (BN / 2 * 128 / 16));
#pragma unroll
                    for (int s4 = 0; s4 < 4; ++s4)
                        mma_ss(go, tmem + S_COL(st), q_d + (uint32_t)(b * (BM * 128 / 16) + s4 * 2), kd + (uint32_t)(s4 * 2),
                               ID_QK, (b > 0 || s4 > 0) ? 1u : 0u);
                    commit(go, k_empty + 8 * k_slot);
                    if (++k_slot == NK) {
                        k_slot = 0;
                        k_phase ^= 1u;
                    }
                }
                commit(go, smem_u32(&sm.s_full[st]));
                if (j == nblk - 1) commit(go, smem_u32(&sm.q_empty));
            };
            while (ok && next_tile()) {
                if (!wait(&sm.q_full, (round - 1) & 1, err, ok)) break;
                issue_s(0);
                if (nblk > 1) issue_s(1);
                for (int j = 0; j < nblk && ok; ++j) {
                    const int st = (g + j) & 1;
                    // the first block's P also says that the last tile's O has been read
                    if (!wait(&sm.p_full[st], ((g + j) >> 1) & 1, err, ok)) break;
#pragma unroll
                    for (int kg = 0; kg < 4; ++kg) {
                        if (!wait(&sm.v_full[v_slot], v_phase, err, ok)) break;
                        fence_after_sync();
                        const uint64_t vd = v_d + (uint64_t)(uint32_t)(v_slot * (32 * 128 * 2 / 16));
#pragma unroll
                        for (int s2 = 0; s2 < 2; ++s2)         // A = P columns of 16 keys
                            mma_ts(go, tmem + O_COL, tmem + S_COL(st) + 8 * (2 * kg + s2), vd + (uint32_t)(s2 * 16 * 128 / 16),
                                   ID_PV, ((LONG ? j % STRETCH : j) > 0 || kg > 0 || s2 > 0) ? 1u : 0u);
                        commit(go, v_empty + 8 * v_slot);
                        if (++v_slot == NV) {
                            v_slot = 0;
                            v_phase ^= 1u;
                        }
                    }
                    commit(go, smem_u32(&sm.pv_done[st]));
                    if (j + 2 < nblk) issue_s(j + 2);
                }
                g += nblk;
            }
        }
    }
    } else if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OUT));
        // ---------------- output: O / l * sigmoid(gate), 32 rows a warp ----------------
        // a lane has 8 dims of a row (f32: 4 of one half); gates are fetched to L2 at the tile's start, to
        // registers AHEAD rows ahead
        constexpr int AHEAD = 8, HALVES = sizeof(T) / 2, DIMS = 8 / HALVES;
        const int r0 = 32 * (warp - 12);
        while (next_tile()) {
            const int rows = (int)max((int64_t)0, min((int64_t)32, tl.T - tl.q0 - r0));   // that exist
            const int64_t first = (tl.row + r0) * nq + qh;             // (row, head) of the first
            for (int i = lane; i < rows * (HD * (int)sizeof(T) / 128); i += 32) {
                constexpr int LINES = HD * (int)sizeof(T) / 128;       // 128-byte lines of a row's gates
                asm volatile("prefetch.global.L2 [%0];" ::"l"(
                    q_gate + (first + (int64_t)(i / LINES) * nq) * QG_ROW + HD + (i % LINES) * (128 / (int)sizeof(T))));
            }
#pragma unroll 1
            for (int half = 0; half < HALVES; ++half) {
                const T* gates = q_gate + first * QG_ROW + HD + 128 * half + DIMS * lane;
                T* to = out + first * HD + 128 * half + DIMS * lane;
                decltype(load4(q_gate)) g0[AHEAD], g1[AHEAD];          // (g1: bf16 only)
                auto load_gates = [&](int i) {
                    const T* p = gates + min(i, rows - 1) * (nq * QG_ROW);
                    g0[i % AHEAD] = load4(p);
                    if (HALVES == 1) g1[i % AHEAD] = load4(p + 4);
                };
                if (rows > 0) {
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) load_gates(i);
                }
                wait(&sm.out_full[half], (round - 1) & 1, err, ok);
#pragma unroll 1
                for (int i0 = 0; ok && i0 < rows; i0 += AHEAD) {
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k) {
                        const int i = i0 + k;
                        const uint4 h = sm.out[r0 + i][lane ^ (i & 7)];
                        const float4 w0 = as_f32(g0[k]), w1 = HALVES == 1 ? as_f32(g1[k]) : w0;
                        load_gates(i + AHEAD);
                        if constexpr (HALVES == 1) {
                            const float2 a = gate2(h.x, w0.x, w0.y), b = gate2(h.y, w0.z, w0.w);
                            const float2 c = gate2(h.z, w1.x, w1.y), e = gate2(h.w, w1.z, w1.w);
                            if (i < rows)
                                store8(to + i * (nq * HD), make_float4(a.x, a.y, b.x, b.y), make_float4(c.x, c.y, e.x, e.y));
                        } else if (i < rows) {
                            *reinterpret_cast<float4*>(to + i * (nq * HD)) = gate4(h, w0);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.out_empty[half]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
        // ---------------- softmax: 8 warps, thread = (query row, key half) ----------------
        const int r = 32 * (warp & 3) + lane;                          // TMEM lane = query row
        const int hf = warp >> 2;                                      // keys [64 hf, 64 hf + 64) of a block
        const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t p_bar[2] = {peer_addr(&sm.p_full[0], 0), peer_addr(&sm.p_full[1], 0)};
        uint32_t g = 0;                                                // blocks so far
        if (LONG) part += (int64_t)blockIdx.x * (BM * HD) + 128 * hf * BM + r;       // this thread's sums
        while (next_tile()) {
            const int64_t qpos = tl.base + tl.q0 + r;                      // absolute position of this query row
            float m_run = -INFINITY, l_run = 0.0f;                         // m identical in both halves; l partial per half
            float m_part = -INFINITY;                                      // m_run when the sums in memory were written
            for (int j0 = 0, j1; j0 < nblk; j0 = j1) {                     // a stretch of blocks
            j1 = LONG ? min(nblk, j0 + STRETCH) : nblk;
            for (int j = j0; j < j1; ++j, ++g) {
                const int st = g & 1;
                // a wait given up (the rest is skipped then, and nothing is stored) leaves no named barrier out
                wait(&sm.s_full[st], (g >> 1) & 1, err, ok);
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
                    for (int c = 4; c < 60; c += 8) {
                        a0 = max3f(a0, s[c], s[c + 1]);
                        a1 = max3f(a1, s[c + 2], s[c + 3]);
                        a2 = max3f(a2, s[c + 4], s[c + 5]);
                        a3 = max3f(a3, s[c + 6], s[c + 7]);
                    }
                    a0 = max3f(a0, s[60], s[61]);
                    a1 = max3f(a1, s[62], s[63]);
                    mx = fmaxf(max3f(a0, a1, a2), a3);
                }
                sm.red_max[st][hf][r] = mx;
                named_bar_sync(1, 256);                                    // also: every S read of this block is done
                mx = fmaxf(mx, sm.red_max[st][hf ^ 1][r]) * q_down;
                const float m_new = fmaxf(m_run, mx);
                const bool grown = m_new > m_run + RESCALE_THRESHOLD;
                if (__any_sync(0xffffffffu, grown)) {
                    // a running max of the warp moved a lot: scale l and this half of the rows of O (by 1
                    // where it did not: TMEM is read and written by whole warps)
                    const float f = grown ? ex2(m_run - m_new) : 1.0f;
                    l_run *= f;
                    if (j > j0) {
                        wait(&sm.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, err, ok);
                        __syncwarp();
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
                    if (grown) m_run = m_new;
                }
                uint32_t pk[32];
                {
                    const uint64_t down = pack2(q_down, q_down), off = pack2(P_LOG2 - m_run, P_LOG2 - m_run);
                    uint64_t acc0 = pack2(0.0f, 0.0f), acc1 = acc0;
#pragma unroll
                    for (int c = 0; c < 64; c += 4) {
                        float x0, x1, p2, p3;
                        unpack2(fma2(pack2(s[c], s[c + 1]), down, off), x0, x1);
                        const float p0 = ex2(x0), p1 = ex2(x1);
                        const uint64_t x23 = fma2(pack2(s[c + 2], s[c + 3]), down, off);
                        if (c % 8 == 0) {                                  // a quarter of them off the special-function unit
                            ex2_poly(x23, p2, p3);
                        } else {
                            float x2, x3;
                            unpack2(x23, x2, x3);
                            p2 = ex2(x2);
                            p3 = ex2(x3);
                        }
                        acc0 = add2(acc0, pack2(p0, p1));
                        acc1 = add2(acc1, pack2(p2, p3));
                        pk[c / 2] = pack_f16(p0, p1);
                        pk[c / 2 + 1] = pack_f16(p2, p3);
                    }
                    float u0, u1;
                    unpack2(add2(acc0, acc1), u0, u1);
                    l_run += u0 + u1;
                }
                // P goes over the first 64 columns of its own S buffer (the previous reader of these
                // columns, PV(j-2), completed before S(j) did)
                tmem_st32(tmem + lane_off + S_COL(st) + 32 * hf, pk);
                fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_at(p_bar[st]);
            }
            if (LONG && j1 < nblk) {                                       // a stretch ends: O to the sums in memory
                wait(&sm.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, err, ok);
                __syncwarp();
                fence_after_sync();
                const float f = ex2(m_part - m_run);
#pragma unroll 1
                for (int c = 0; c < 128; c += 16) {                        // (by 32 the f32 kernel took a quarter longer)
                    uint32_t o[16];
                    tmem_ld16_async(tmem + lane_off + O_COL + 128 * hf + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float* sum = part + (c + i) * BM;
                        *sum = fmaf(j0 > 0 ? *sum : 0.0f, f, __uint_as_float(o[i]));
                    }
                }
                m_part = m_run;
                fence_before_sync();
            }
            }
            // O / l of this thread's row, dims [128 hf, 128 hf + 128), to the output warps
            sm.red_l[hf][r] = l_run;
            named_bar_sync(1, 256);
            constexpr bool F32 = sizeof(T) == 4;
            const float inv_l = (F32 ? 1.0f : OUT_SCALE) / (l_run + sm.red_l[hf ^ 1][r]);
            // the place is free: from the last tile's rows, or (f32) their second half, or this tile's first
            if (round > 1 && !(F32 && hf == 1)) wait(&sm.out_empty[F32], round & 1, err, ok);
            if (F32 && hf == 1) wait(&sm.out_empty[0], (round - 1) & 1, err, ok);
            wait(&sm.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, err, ok);
            __syncwarp();
            fence_after_sync();
            if (LONG && nblk > STRETCH) {                                  // and the sums in memory, into TMEM
                const float f = ex2(m_part - m_run);
#pragma unroll 1
                for (int c = 0; c < 128; c += 16) {
                    uint32_t o[16];
                    tmem_ld16_async(tmem + lane_off + O_COL + 128 * hf + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(fmaf(part[(c + i) * BM], f, __uint_as_float(o[i])));
                    tmem_st16(tmem + lane_off + O_COL + 128 * hf + c, o);
                }
            }
#pragma unroll
            for (int c0 = 0; c0 < 128; c0 += 32) {
                float o[32];
                tmem_ld32(tmem + lane_off + O_COL + 128 * hf + c0, o);
                if constexpr (F32) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        sm.out[r][((c0 + i) / 4) ^ (r & 7)] =
                            make_uint4(__float_as_uint(o[i] * inv_l), __float_as_uint(o[i + 1] * inv_l),
                                       __float_as_uint(o[i + 2] * inv_l), __float_as_uint(o[i + 3] * inv_l));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        sm.out[r][((128 * hf + c0 + i) / 8) ^ (r & 7)] =
                            make_uint4(pack_f16(o[i] * inv_l, o[i + 1] * inv_l), pack_f16(o[i + 2] * inv_l, o[i + 3] * inv_l),
                                       pack_f16(o[i + 4] * inv_l, o[i + 5] * inv_l), pack_f16(o[i + 6] * inv_l, o[i + 7] * inv_l));
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.out_full[F32 ? hf : 0]);
        }
    }
    // neither CTA leaves, or frees TMEM, while the other's products or arrivals may touch it; after
    // a wait that was given up, copies and products already issued get time to end
    if (!ok) settle();
    fence_before_sync();
    __syncthreads();
    cluster_sync();
    if (warp == 0) dealloc(tmem, 512);
}

// f16 tensor [d2][d1][256] with a (64 x rows x 1) box, 128-byte swizzle
static bool make_map(CUtensorMap* m, const void* base, int64_t d1, int64_t d2, int box_rows) {
    const EncodeTiledFn fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)d1, (cuuint64_t)d2};
    const cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)d1 * HD * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace attn
}  // namespace q4

cudaError_t q4_prefill_setup() {
    using B = __nv_bfloat16;
    cudaError_t e = cudaSuccess;
    using namespace q4::attn;
    for (auto kernel : {(const void*)q4_pf_attn_kernel<float, false>, (const void*)q4_pf_attn_kernel<float, true>,
                        (const void*)q4_pf_attn_kernel<B, false>, (const void*)q4_pf_attn_kernel<B, true>})
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    return e;
}

// The attention CTAs' sums in memory, where a sequence has more than a stretch of keys.
static int64_t part_bytes(const dz_ctx* ctx, const q4::Prompt& d) {
    int longest = 0;
    for (int s = 0; s < d.n; ++s) longest = std::max(longest, d.key0[s + 1] - d.key0[s]);
    return longest > q4::attn::STRETCH * q4::attn::BN ? ctx->n_sm * q4::attn::PART_BYTES : 0;
}

template <typename T>
static cudaError_t launch_group(dz_ctx* ctx, int layer, const q4::Prompt& d, const int32_t* pos, const T* q_gate,
                                const T* k, const T* v, T* out, cudaStream_t st, int* n_launch) {
    const LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
    const int64_t tokens = d.row0[d.n], keys = d.key0[d.n];
    const size_t qn = (size_t)nq * tokens * HD, kn = (size_t)kvc * keys * HD;
    cudaError_t e;
    __half* qf = static_cast<__half*>(ctx->q4_scratch);
    __half *kf = qf + qn, *vf = kf + kn;
    float* part = reinterpret_cast<float*>(vf + kn);           // behind them where a sequence needs it (part_bytes)
    CUtensorMap mq, mk, mv;
    using namespace q4;
    if (!attn::make_map(&mq, qf, tokens, nq, attn::BM) || !attn::make_map(&mk, kf, keys, kvc, attn::BN / 2) ||
        !attn::make_map(&mv, vf, keys, kvc, 32))
        return cudaErrorInvalidValue;
    attn::Packed map;
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
        map.first[i + 1] = map.first[i] + attn::Packed::own_tiles(d.T(s), map.split_idx, map.split_cnt);
    }
    // Heads that share a warp's set-up (positions, angles, weights): half of them, and a tile's kv heads,
    // where that leaves 20 warps per SM, else 4 and one (the call with 1000 tokens: 37 us, 42 with half
    // and all; with 1500: 56 and 55; with 2000 after 5555: 246 and 240).
    const bool many = tokens >= 10 * (int64_t)ctx->n_sm;
    const int q_heads = many ? nq / 2 : PREP_ROWS, key_heads = many ? kvc : 1;
    const int64_t q_tasks = tokens * ((nq + q_heads - 1) / q_heads);
    const int64_t blocks = (int64_t)d.at0[d.n] * (kvc / key_heads) + (int64_t)d.old0[d.n] * kvc +
                           (q_tasks + PREP_WARPS - 1) / PREP_WARPS;
    q4_pf_prep_kernel<T><<<(unsigned)blocks, 32 * PREP_WARPS, 0, st>>>(
        d, ctx->axes, kvc, L.d_q4, pos, L.q_norm, L.k_norm, q_gate, k, v, qf, kf, vf, key_heads, q_heads, ctx->q4_track,
        ctx->cfg.rms_eps, L.q_up);
    *n_launch += 1;
    if (map.first[d.n] > 0) {
        const unsigned clusters = (unsigned)std::min((int64_t)map.first[d.n] * nq / 2, (int64_t)ctx->n_sm / 2);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t lc{};
        lc.gridDim = dim3(2 * clusters);
        lc.blockDim = dim3(attn::NTHREADS);
        lc.dynamicSmemBytes = attn::SMEM_BYTES;
        lc.stream = st;
        lc.attrs = at;
        lc.numAttrs = 1;
        auto kernel = part_bytes(ctx, d) > 0 ? attn::q4_pf_attn_kernel<T, true> : attn::q4_pf_attn_kernel<T, false>;
        e = cudaLaunchKernelEx(&lc, kernel, mq, mk, mv, map, kvc, q_gate, out, part, 1.0f / L.q_up, ctx->d_err);
        if (e != cudaSuccess) return e;
        *n_launch += 1;
    }
    return cudaGetLastError();
}

// Sequences are taken in groups whose scratch (f16 queries, keys and values) stays below
// this, unless one alone is larger.
static constexpr int64_t GROUP_BYTES = (int64_t)2 << 30;

// The group that begins at sequence i (i moves behind it); its scratch in bytes, 0 if no tokens are left.
static int64_t next_group(const LayerState& L, int kvc, int& i, int n, const int32_t* seq_ids, const int64_t* lens,
                          q4::Prompt& d) {
    d.n = 0;
    d.row0[0] = d.key0[0] = d.at0[0] = d.old0[0] = 0;
    int64_t bytes = 0;
    for (; i < n && d.n < MAXB; ++i) {
        const int64_t base = L.len[seq_ids[i]], T_i = lens[i];
        const int64_t keys = (base + T_i + q4::attn::BN - 1) / q4::attn::BN * q4::attn::BN;
        const int64_t more = (T_i * GRP + 2 * keys) * kvc * HD * (int64_t)sizeof(__half);
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
    return bytes;
}

// All or nothing: scratch for the largest group before the first launch, lengths after the last.
template <typename T>
static cudaError_t launch_prompts(dz_ctx* ctx, int layer, int n, const int32_t* seq_ids, const int64_t* lens,
                                  const int32_t* pos, const T* q_gate, const T* k, const T* v, T* out, cudaStream_t st,
                                  int* n_launch) {
    LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count, nq = GRP * kvc;
    q4::Prompt d;
    int64_t most = 0;
    for (int i = 0; i < n;) {
        const int64_t bytes = next_group(L, kvc, i, n, seq_ids, lens, d);
        most = std::max(most, bytes + part_bytes(ctx, d));
    }
    cudaError_t e = ensure_q4_scratch(ctx, most);
    if (e != cudaSuccess) return e;
    for (int i = 0; i < n;) {
        if (next_group(L, kvc, i, n, seq_ids, lens, d) == 0) break;
        if ((e = launch_group<T>(ctx, layer, d, pos, q_gate, k, v, out, st, n_launch)) != cudaSuccess) return e;
        const size_t rows = d.row0[d.n];
        if (pos) pos += 3 * rows;
        q_gate += rows * nq * QG_ROW;
        k += rows * kvc * HD;
        v += rows * kvc * HD;
        out += rows * nq * HD;
    }
    for (int i = 0; i < n; ++i) L.len[seq_ids[i]] += lens[i];
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
