// q4_decode.cu -- split-K decode attention over the 4-bit KV cache (q4.cuh).
//
// The gated GQA core of attention.rs:90-203 for one token per sequence, with K and V
// held in 4 bits and rotary positions of three axes.  Stream-ordered kernels:
//   1. q4_prep     : per sequence and head -- deinterleave [Q_h | gate_h], QK-RMSNorm,
//                    rotation; q as matrix operand, K and V quantised into slot len.
//   2. q4_split    : scores, online softmax and P V over the cached tiles, cut evenly
//                    over the SMs; unnormalised partials out.
//   3. q4_combine  : per (sequence, q head) -- merge, normalise, gate; tracked caches: further
//                    blocks add the new attention weights.
// One call, 24 q heads on 4 kv heads: one sequence of 2048, 10.4 us (three dependent grids:
// latency); 64 of 512-32768 (1.17 GB), 294 us, 3.98 TB/s; 8 of 131072 (1.14 GB), 275 us,
// 4.15 TB/s, 0.63 of a plain copy's rate.
#include <algorithm>
#include <cstddef>

#include "q4.cuh"

namespace dz {
namespace q4 {

// ---------------------------------------------------------------------------
// 1. prep: grid (B, ceil((nq + kvc) / 8)), one head per warp.
//    q is scaled by log2(e) (scores in log2 units; the 1/16 comes with K's unpacking,
//    which gives K / 16) and by a power of two that
//    puts the head's largest magnitude into [2^11, 2^12), then split into f16 hi + lo
//    (22 bits; f16 subnormals start 2^25 below), in the register order of the A
//    operand of mma.m16n8k16: rows 0..7 are the hi parts of the group's heads (6 and 7
//    empty), rows 8..15 the lo parts, so one product of K gives both.
//      q_frag [b][kvh][step 16][lane][hi 0,1 | lo 0,1 | hi 2,3 | lo 2,3]
//    where step s, lane (r, c) covers dims 64 c + 4 s .. + 3 of head r.
//    and behind the 16 steps the heads' factors back (f32 [8], 0 for the empty heads).
//    K goes through f32 first (quantise_key): with f64 throughout, the call for one
//    sequence took 13.0 us.  Running this inside the split grid (each CTA its own rows)
//    was slower: 64 CTAs of few sequences wait for it as for a grid.
// ---------------------------------------------------------------------------
using Rows = Q4Rows;
constexpr int FRAG_WORDS = Q4_FRAG_WORDS, FRAG_SCALES = 16 * 32 * 4;

__global__ void __launch_bounds__(256) q4_prep_kernel(const __grid_constant__ Rows d, const __grid_constant__ Q4Pos pos,
                                                      RopeAxes axes, const Q4Slot* __restrict__ slots,
                                                      const float* __restrict__ q_norm, const float* __restrict__ k_norm,
                                                      const float* __restrict__ q_gate, const float* __restrict__ k_in,
                                                      const float* __restrict__ v_in, uint32_t* __restrict__ q_frag,
                                                      float eps) {
    __shared__ double2 cs[8][ROPE / 2];
    __shared__ float2 csf[8][ROPE / 2];
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvc = d.kvc, nq = GRP * kvc;
    const int task = blockIdx.y * 8 + warp;
    // before the wait: the angles
    csf[warp][lane] = rope_cs_f32(axes, lane, pos.p[b][0], pos.p[b][1], pos.p[b][2]);
    __syncwarp();
    // As in gqa_prep: everything before this grid is complete (inputs, caches, q_frag)
    // before the split grid may start streaming old tiles.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (task >= nq + kvc) return;
    if (task < nq) {
        const float4* src = reinterpret_cast<const float4*>(q_gate + ((size_t)b * nq + task) * QG_ROW);
        const float4 a0 = src[2 * lane], a1 = src[2 * lane + 1];
        float x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
        norm_rotate(x, q_norm, csf[warp], eps, lane);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] *= LOG2E;
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
        if (lane == 0) reinterpret_cast<uint32_t*>(dst)[FRAG_SCALES + r] = (uint32_t)(254 - field) << 23;
    } else {
        const int kvh = task - nq, slot_pos = d.len[b];
        uint4* dst = reinterpret_cast<uint4*>(q_frag + (size_t)(b * kvc + kvh) * FRAG_WORDS);
#pragma unroll
        for (int i = 0; i < 4; ++i)                            // the operand's empty rows: heads 6 and 7
            dst[(4 * i + (lane >> 3)) * 32 + 24 + (lane & 7)] = make_uint4(0u, 0u, 0u, 0u);
        if (lane < 2) reinterpret_cast<uint32_t*>(dst)[FRAG_SCALES + 6 + lane] = 0u;
        uint8_t* tile = slots[d.sid[b]].tile(kvh, slot_pos >> 4);
        const int p = slot_pos & 15;
        const size_t at = ((size_t)b * kvc + kvh) * HD + 8 * lane;
        const float4 k0 = *reinterpret_cast<const float4*>(k_in + at), k1 = *reinterpret_cast<const float4*>(k_in + at + 4);
        const float4 v0 = *reinterpret_cast<const float4*>(v_in + at), v1 = *reinterpret_cast<const float4*>(v_in + at + 4);
        const float x[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
        float y[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        uint32_t code[8];
        uint32_t sb = quantise_key(x, k_norm, csf[warp], cs[warp], axes, pos.p[b][0], pos.p[b][1], pos.p[b][2], eps,
                                   lane, code);
        put_k(tile, p, lane, code, sb);
        sb = quantise(y, code);
        uint4* vw = v_words(tile, lane, (p & 7) >> 1);
        uint4 w = *vw;
        merge_v(w, p, code);
        *vw = w;
        put_v_scale(tile, p, lane, sb);
    }
}

// ---------------------------------------------------------------------------
// 2. attention over the tiles, the whole batch cut into equal runs of tiles, a warp each.
//    Rows are (sequence, kv head) in order; their tiles are numbered through, and run c
//    of R takes tiles [W c / R, W (c + 1) / R): every warp reads the same number of bytes
//    however ragged the batch is, and no warp waits for another.  A run covers parts of
//    one or more rows; each part (segment) gives one unnormalised partial, at index
//    c + row (unique: both only grow along the runs).
//    Tiles come in pairs (32 positions, 8704 bytes): one bulk copy into the warp's own
//    ring, requested across segment ends.
//    Scores: S = Q K^T, A = q (hi rows, lo rows; in registers), B = the 8 positions of a K word row, 16
//    steps of 16 dims; thread (r, c) gets head r at positions 2c, 2c+1 (hi sum and lo sum,
//    added).  That is the B operand's own layout, so P needs no shuffle: O^T += V^T P^T,
//    A = V's dims x 16 positions, B = P (hi, then lo), 16 tiles of 16 dims accumulated in
//    64 registers.
//    Bound by issue: the 64 matrix instructions of a tile take 131 cycles of an SM (a
//    sub-core is held 8 cycles by each), unpacking, softmax and sums bring it to 235; the
//    tile's bytes take 189 at the copy rate.  tcgen05 would want the codes unpacked into
//    shared memory for 6 of 128 rows.  8 warps with 255 registers: 12 with 168 kept q in
//    shared memory, and 64 sequences took 342 us; e4m3 products (a conversion and two f16
//    products on this GPU) were slower still; adding partial sums of single tiles instead of
//    pairs: 315 us.  Equal runs of tiles per warp against per CTA: 285 and 303 us with the
//    12 warps.
// ---------------------------------------------------------------------------
constexpr int STAGES = 3, WARPS = 8;
// p is taken against a maximum that may be stale by P_SLACK and is scaled by 2^P_LOG2: at
// most 2^15, and its f16 lo part keeps its bits down to 2^-21 of the maximum.
constexpr float P_LOG2 = 8.0f, P_SLACK = 7.0f;

struct alignas(128) Ring {
    uint8_t pair[STAGES][2 * Q4_TILE_BYTES];
    uint64_t full[STAGES];
};
constexpr int SPLIT_SMEM = WARPS * (int)sizeof(Ring);
static_assert(Q4_TILE_BYTES % 128 == 0 && sizeof(Ring) % 128 == 0, "bulk copies need 16-byte alignment");

// Run c starts at tile c * run_base + min(c, run_rem) (tiles = runs * run_base + run_rem).
__host__ __device__ inline int run_start(const Rows& d, int c) { return c * d.run_base + min(c, d.run_rem); }
// the run that holds a tile
__device__ __forceinline__ int run_of(const Rows& d, int tile) {
    const int longer = d.run_rem * (d.run_base + 1);           // tiles of the runs that have one more
    return tile < longer ? (int)((uint32_t)tile / (uint32_t)(d.run_base + 1))
                         : d.run_rem + (int)((uint32_t)(tile - longer) / (uint32_t)d.run_base);
}

// The part of a row that a run covers: tiles [t0, t1) of the row.
struct Segment { int b, row, t0, t1; const uint8_t* base; };

__device__ __forceinline__ Segment segment_at(const Rows& d, const Q4Slot* __restrict__ slots, int tile, int end) {
    Segment s;
    int lo = 0, hi = d.B - 1;                    // last b whose rows start at or before the tile
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (d.cum[mid] * d.kvc <= tile) lo = mid; else hi = mid - 1;
    }
    s.b = lo;
    const int n = d.row_tiles(lo);
    int in = tile - d.cum[lo] * d.kvc, kvh = 0;
    while (in >= n) {
        in -= n;
        ++kvh;
    }
    s.row = lo * d.kvc + kvh;
    s.t0 = in;
    s.t1 = min(n, in + (end - tile));
    s.base = slots[d.sid[lo]].tile(kvh, 0);
    return s;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same from 0
__device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// f32 pairs: a += (x, y)
__device__ __forceinline__ void add2(uint64_t& a, float x, float y) {
    asm("{.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;}" : "+l"(a) : "f"(x), "f"(y));
}
__device__ __forceinline__ float2 halves(uint64_t a) {
    float2 d;
    unpack2(a, d.x, d.y);
    return d;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One warp's running softmax over the tiles that it takes of a segment.
struct State {
    uint64_t o[16][2];                           // O^T / 16: tile m, dims 32 r + 2 m, + 1: pair of heads 2c, 2c + 1
    float m, l;                                  // head r; l is this thread's share
};

// NT tiles (1 or 2).  valid: positions of them that exist.
template <int NT, bool TRACK>
__device__ __forceinline__ void attend(State& st, const uint8_t* tiles, const uint4 (&q)[16], float qs, int valid,
                                       float* __restrict__ scores, int lane) {
    const int r = lane >> 2, c = lane & 3;
    // ---- scores of NT x 2 x 8 positions: x[n][0], x[n][1] = head r at positions 8 n + 2 c, + 1
    float x[2 * NT][2];
    {
        float s[2 * NT][4] = {};                 // hi and lo sums
        uint32_t kb[NT];
#pragma unroll
        for (int k = 0; k < NT; ++k)
            kb[k] = *reinterpret_cast<const uint32_t*>(tiles + k * Q4_TILE_BYTES + OFF_KS + lane * 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t ws[2 * NT][4];
            Scale16 sc[2 * NT];
#pragma unroll
            for (int n = 0; n < 2 * NT; ++n) {
                const uint4 w4 = *reinterpret_cast<const uint4*>(tiles + (n >> 1) * Q4_TILE_BYTES + ((n & 1) * 2 + i) * 512 +
                                                                 lane * 16);
                ws[n][0] = w4.x; ws[n][1] = w4.y; ws[n][2] = w4.z; ws[n][3] = w4.w;
                // the group's scale byte in both halves
                sc[n] = scale16(scale_pair(__byte_perm(kb[n >> 1], 0u, 0x4040 + 0x0101 * ((n & 1) * 2 + i))));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint4 qa = q[8 * i + 2 * u], qb = q[8 * i + 2 * u + 1];
#pragma unroll
                for (int n = 0; n < 2 * NT; ++n)
                    mma(s[n], qa.x, qa.y, qa.z, qa.w, unpack_lo(ws[n][u], sc[n]), unpack_hi(ws[n][u], sc[n]));
#pragma unroll
                for (int n = 0; n < 2 * NT; ++n) {
                    const uint32_t w8 = ws[n][u] >> 8;
                    mma(s[n], qb.x, qb.y, qb.z, qb.w, unpack_lo(w8, sc[n]), unpack_hi(w8, sc[n]));
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) {
            x[n][0] = (s[n][0] + s[n][2]) * qs;
            x[n][1] = (s[n][1] + s[n][3]) * qs;
        }
    }
    if (TRACK) {
        if (r < GRP) {                           // [tile][head][16]
#pragma unroll
            for (int n = 0; n < 2 * NT; ++n)
                *reinterpret_cast<float2*>(scores + ((n >> 1) * GRP + r) * Q4_TILE + 2 * c + 8 * (n & 1)) =
                    make_float2(x[n][0], x[n][1]);
        }
    }
    if (valid < NT * Q4_TILE) {                  // the row's last tile
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) {
            if (8 * n + 2 * c >= valid) x[n][0] = -INFINITY;
            if (8 * n + 2 * c + 1 >= valid) x[n][1] = -INFINITY;
        }
    }
    // ---- online softmax
    float mx = fmaxf(x[0][0], x[0][1]);
#pragma unroll
    for (int n = 1; n < 2 * NT; ++n) mx = fmaxf(mx, fmaxf(x[n][0], x[n][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // rescale only when some head's maximum has outgrown what f16 holds of 2^P_LOG2 p
    if (__any_sync(0xffffffffu, mx > st.m + P_SLACK)) {
        const float m_new = fmaxf(st.m, mx), a = ex2f(st.m - m_new);
        st.l *= a;
        st.m = m_new;
        const float a0 = __shfl_sync(0xffffffffu, a, 8 * c), a1 = __shfl_sync(0xffffffffu, a, 8 * c + 4);
        const uint64_t aa = pack2(a0, a1);
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            st.o[m][0] = mul2(st.o[m][0], aa);
            st.o[m][1] = mul2(st.o[m][1], aa);
        }
    }
    const float off = P_LOG2 - st.m;
    uint32_t ph[2 * NT], pl[2 * NT];
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n) {
        const float p0 = ex2f(x[n][0] + off), p1 = ex2f(x[n][1] + off);
        st.l += p0 + p1;
        const __half2 h = __floats2half2_rn(p0, p1);
        const __half2 l = __floats2half2_rn(p0 - __low2float(h), p1 - __high2float(h));
        ph[n] = *reinterpret_cast<const uint32_t*>(&h);
        pl[n] = *reinterpret_cast<const uint32_t*>(&l);
    }
    // ---- O^T += V^T P^T.  The matrix instruction adds to its f32 accumulator with truncation
    // (n additions leave it about n 2^-24 short: 5e-6 over 148 tiles when O was the
    // accumulator), so the tiles' product starts from 0 and is added to O rounded to nearest.
    Scale16 sa[NT], sb[NT];
#pragma unroll
    for (int k = 0; k < NT; ++k) {
        const uint32_t vb = *reinterpret_cast<const uint32_t*>(tiles + k * Q4_TILE_BYTES + OFF_VS + lane * 4);
        sa[k] = scale16(scale_pair(__byte_perm(vb, 0u, 0x4140)));
        sb[k] = scale16(scale_pair(__byte_perm(vb, 0u, 0x4342)));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float d[4][4];
#pragma unroll
        for (int k = 0; k < NT; ++k) {
            const uint4 w4 = *reinterpret_cast<const uint4*>(tiles + k * Q4_TILE_BYTES + v_at(i, r, c));
            const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t w = ws[u], w8 = w >> 8;
                const uint32_t a0 = unpack_lo(w, sa[k]), a2 = unpack_hi(w, sb[k]);
                const uint32_t a1 = unpack_lo(w8, sa[k]), a3 = unpack_hi(w8, sb[k]);
                if (k == 0) mma0(d[u], a0, a1, a2, a3, ph[0], ph[1]);
                else mma(d[u], a0, a1, a2, a3, ph[2 * k], ph[2 * k + 1]);
                mma(d[u], a0, a1, a2, a3, pl[2 * k], pl[2 * k + 1]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            add2(st.o[4 * i + u][0], d[u][0], d[u][1]);
            add2(st.o[4 * i + u][1], d[u][2], d[u][3]);
        }
    }
}

template <bool TRACK>
__global__ void __launch_bounds__(32 * WARPS, 1)
    q4_split_kernel(const __grid_constant__ Rows d, const Q4Slot* __restrict__ slots,
                    const uint32_t* __restrict__ q_frag, float* __restrict__ part_o, float* __restrict__ part_ml,
                    float* __restrict__ scores, int* err) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    Ring& ring = reinterpret_cast<Ring*>(smem_raw)[warp];
    asm volatile("griddepcontrol.launch_dependents;");
    const int run = warp * gridDim.x + blockIdx.x;   // few runs: spread over the SMs first
    if (run >= d.runs) return;
    const int run0 = run_start(d, run), run1 = run_start(d, run + 1);
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&ring.full[s], 1);
        fence_mbar_init();
    }
    __syncwarp();
    // producer: the next tile to request
    int p_end = run0;                        // end of the producer's segment
    Segment ps{};
    int p_t = 0;
    // the tile that holds slot len is written by q4_prep: requested after the grid-dependency wait
    bool dep_done = false;
    auto wait_prep = [&]() {
        if (!dep_done) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            dep_done = true;
        }
    };
    auto produce = [&](int stage) {
        if (p_t == ps.t1) {
            if (p_end == run1) return;
            ps = segment_at(d, slots, p_end, run1);
            p_end += ps.t1 - ps.t0;
            p_t = ps.t0;
        }
        const int nt = min(2, ps.t1 - p_t);
        if (p_t + nt == d.row_tiles(ps.b)) wait_prep();
        if (lane == 0) {
            mbar_arrive_expect_tx(&ring.full[stage], nt * Q4_TILE_BYTES);
            bulk_g2s(ring.pair[stage], ps.base + (size_t)p_t * Q4_TILE_BYTES, nt * Q4_TILE_BYTES, &ring.full[stage]);
        }
        p_t += nt;
    };
    for (int s = 0; s < STAGES; ++s) produce(s);
    wait_prep();                                 // q_frag

    int stage = 0;
    uint32_t phase = 0;
    for (int at = run0; at < run1;) {
        const Segment sg = segment_at(d, slots, at, run1);
        const uint32_t* frag = q_frag + (size_t)sg.row * FRAG_WORDS;
        uint4 q[16];
#pragma unroll
        for (int s = 0; s < 16; ++s) q[s] = reinterpret_cast<const uint4*>(frag)[s * 32 + lane];
        const float qs = __uint_as_float(frag[FRAG_SCALES + r]);
        const int n = d.len[sg.b] + 1;
        State st;
#pragma unroll
        for (int m = 0; m < 16; ++m) st.o[m][0] = st.o[m][1] = 0ull;
        st.m = -INFINITY;
        st.l = 0.0f;
        for (int t = sg.t0; t < sg.t1; t += 2) {
            // given up: the warp's other copies, all issued before, have had the whole limit to end
            if (!mbar_wait(&ring.full[stage], phase, err)) return;
            float* sc = TRACK ? scores + (size_t)(at + (t - sg.t0)) * (GRP * Q4_TILE) : nullptr;
            if (t + 1 < sg.t1) attend<2, TRACK>(st, ring.pair[stage], q, qs, n - t * Q4_TILE, sc, lane);
            else attend<1, TRACK>(st, ring.pair[stage], q, qs, n - t * Q4_TILE, sc, lane);
            __syncwarp();
            produce(stage);
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
        at += sg.t1 - sg.t0;
        // ---- the segment's partial: thread (r, c) holds dims 32 r .. + 31 of heads 2c, 2c + 1
        st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
        st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
        const size_t part = (size_t)run + sg.row;
        if (c < GRP / 2) {
            float* po = part_o + (part * GRP + 2 * c) * HD + 32 * r;
#pragma unroll
            for (int m = 0; m < 16; m += 2) {    // V came as V / 16
                const float2 a0 = halves(st.o[m][0]), b0 = halves(st.o[m][1]);
                const float2 a1 = halves(st.o[m + 1][0]), b1 = halves(st.o[m + 1][1]);
                *reinterpret_cast<float4*>(po + 2 * m) = make_float4(16.0f * a0.x, 16.0f * b0.x, 16.0f * a1.x, 16.0f * b1.x);
                *reinterpret_cast<float4*>(po + HD + 2 * m) =
                    make_float4(16.0f * a0.y, 16.0f * b0.y, 16.0f * a1.y, 16.0f * b1.y);
            }
        }
        if (c == 0 && r < GRP)
            reinterpret_cast<float2*>(part_ml)[part * GRP + r] = make_float2(st.m - P_LOG2, st.l);
    }
}

// ---------------------------------------------------------------------------
// 3. tracked caches: weight of position j of a kv head += sum over its 6 q heads of
//    exp2(score - M) / L, with M and L merged from the partials' (m, l).  The new
//    position's weight starts here.  A block takes WT_SPAN positions of a (sequence, kv head).
//    In the combine grid, beside its blocks: 12 sequences of 1137-7414 take 34.5 us (30 without
//    weights; 38 as a kernel of its own behind it; 35.0 and 34.7 with spans of 1024 and 256).
// ---------------------------------------------------------------------------
constexpr int WT_SPAN = 512;

__device__ __forceinline__ void add_weights(const Rows& d, int b, int kvh, int span, const Q4Slot* __restrict__ slots,
                                            const float* __restrict__ part_ml, const float* __restrict__ scores) {
    __shared__ float M[GRP], L[GRP];
    const int n = d.len[b] + 1, j0 = span * WT_SPAN;
    if (j0 >= n) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = b * d.kvc + kvh;
    const int start = d.row_start(row), c0 = run_of(d, start), nc = run_of(d, start + d.row_tiles(b) - 1) - c0 + 1;
    const Q4Slot slot = slots[d.sid[b]];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp < GRP) {
        const float2* ml = reinterpret_cast<const float2*>(part_ml) + ((size_t)c0 + row) * GRP + warp;
        float m = -INFINITY;
        for (int i = lane; i < nc; i += 32) m = fmaxf(m, ml[(size_t)i * GRP].x);
        m = warp_max(m);
        float l = 0.0f;
        for (int i = lane; i < nc; i += 32) {
            const float2 v = ml[(size_t)i * GRP];
            l += v.y * exp2f(v.x - m);
        }
        l = warp_sum(l);
        if (lane == 0) {
            M[warp] = m;
            L[warp] = 1.0f / l;
        }
    }
    __syncthreads();
    float* wts = slot.wts + (size_t)kvh * slot.cap;
    for (int j = j0 + threadIdx.x; j < min(n, j0 + WT_SPAN); j += 256) {
        const float* sc = scores + (size_t)(start + (j >> 4)) * (GRP * Q4_TILE) + (j & 15);
        float w = 0.0f;
#pragma unroll
        for (int h = 0; h < GRP; ++h) w += ex2f(sc[h * Q4_TILE] - M[h]) * L[h];
        wts[j] = w + (j < n - 1 ? wts[j] : 0.0f);
    }
}

// ---------------------------------------------------------------------------
// 4. combine: merge a row's partials, divide, gate.  Grid (6 kvc x 4 quarters of the
//    dims, then the blocks of the weights; B), 16 groups of 16 threads that take partials in turn, 4 dims a thread.  Latency:
//    about 3 us of a call.
// ---------------------------------------------------------------------------
constexpr int MAX_RUNS = 2048;                   // warps of the split grid (148 SMs: 1184)
constexpr int CMB_DIMS = 64;

template <bool TRACK>
__global__ void __launch_bounds__(256) q4_combine_kernel(const __grid_constant__ Rows d,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ part_ml,
                                                         const float* __restrict__ q_gate, float* __restrict__ out,
                                                         const Q4Slot* __restrict__ slots,
                                                         const float* __restrict__ scores) {
    __shared__ float wgt[MAX_RUNS];
    __shared__ float red[2][8];
    __shared__ float4 acc[16][CMB_DIMS / 4];
    asm volatile("griddepcontrol.launch_dependents;");
    const int nq = GRP * d.kvc, b = blockIdx.y, quarter = blockIdx.x / nq, tid = threadIdx.x;
    const int qh = blockIdx.x - quarter * nq, d0 = quarter * CMB_DIMS;
    if (TRACK && quarter >= HD / CMB_DIMS) {
        const int at = blockIdx.x - HD / CMB_DIMS * nq;
        add_weights(d, b, at % d.kvc, at / d.kvc, slots, part_ml, scores);
        return;
    }
    const int kvh = qh / GRP, h = qh - kvh * GRP, row = b * d.kvc + kvh;
    const int warp = tid >> 5, lane = tid & 31;
    const float gate = tid < CMB_DIMS ? q_gate[((size_t)b * nq + qh) * QG_ROW + HD + d0 + tid] : 0.0f;
    const int start = d.row_start(row), c0 = run_of(d, start), nc = run_of(d, start + d.row_tiles(b) - 1) - c0 + 1;
    const size_t part0 = (size_t)c0 + row;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float2* ml = reinterpret_cast<const float2*>(part_ml) + part0 * GRP + h;
    float m = -INFINITY;
    for (int i = tid; i < nc; i += 256) m = fmaxf(m, ml[(size_t)i * GRP].x);
    m = warp_max(m);
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    float M = red[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) M = fmaxf(M, red[0][w]);
    float l = 0.0f;
    for (int i = tid; i < nc; i += 256) {
        const float2 v = ml[(size_t)i * GRP];
        const float w = exp2f(v.x - M);
        wgt[i] = w;
        l += v.y * w;
    }
    l = warp_sum(l);
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    const int g = tid >> 4, e = tid & 15;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = g; i < nc; i += 16) {
        const float4 v = reinterpret_cast<const float4*>(part_o + ((part0 + i) * GRP + h) * HD + d0)[e];
        const float w = wgt[i];
        a.x = fmaf(v.x, w, a.x);
        a.y = fmaf(v.y, w, a.y);
        a.z = fmaf(v.z, w, a.z);
        a.w = fmaf(v.w, w, a.w);
    }
    acc[g][e] = a;
    __syncthreads();
    if (tid < CMB_DIMS) {
        float L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) L += red[1][w];
#pragma unroll
        for (int k = 0; k < 16; ++k) o += reinterpret_cast<const float*>(acc[k])[tid];
        out[((size_t)b * nq + qh) * HD + d0 + tid] = o * (1.0f / L) * sigmoidf_acc(gate);
    }
}

}  // namespace q4

cudaError_t q4_decode_setup() {
    const cudaError_t e = cudaFuncSetAttribute(q4::q4_split_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               q4::SPLIT_SMEM);
    return e != cudaSuccess ? e
                            : cudaFuncSetAttribute(q4::q4_split_kernel<true>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, q4::SPLIT_SMEM);
}

int q4_decode_runs(int n_sm) { return std::min(q4::WARPS * n_sm, q4::MAX_RUNS); }

cudaError_t launch_q4_decode(dz_ctx* ctx, int layer, Q4Rows& d, const Q4Pos& pos, const float* q_gate,
                             const float* k, const float* v, float* out, cudaStream_t st, int* n_launch) {
    using namespace q4;
    const LayerState& L = ctx->layers[layer];
    const int kvc = d.kvc;
    d.runs = std::min(d.tiles(), q4_decode_runs(ctx->n_sm));
    d.run_base = d.tiles() / d.runs;
    d.run_rem = d.tiles() % d.runs;
    auto split = ctx->q4_track ? q4_split_kernel<true> : q4_split_kernel<false>;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(d.B, (GRP * kvc + kvc + 7) / 8);
    lc.blockDim = dim3(256);
    lc.stream = st;
    lc.attrs = at;
    lc.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&lc, q4_prep_kernel, d, pos, ctx->axes, (const Q4Slot*)L.d_q4, (const float*)L.q_norm,
                           (const float*)L.k_norm, q_gate, k, v, ctx->q4_frag, ctx->cfg.rms_eps);
    if (e != cudaSuccess) return e;
    lc.gridDim = dim3(std::min(d.runs, ctx->n_sm));
    lc.blockDim = dim3(32 * WARPS);
    lc.dynamicSmemBytes = SPLIT_SMEM;
    e = cudaLaunchKernelEx(&lc, split, d, (const Q4Slot*)L.d_q4, (const uint32_t*)ctx->q4_frag, ctx->part_o,
                           ctx->part_ml, ctx->q4_sc, ctx->d_err);
    if (e != cudaSuccess) return e;
    int blocks = GRP * kvc * (HD / CMB_DIMS);
    if (ctx->q4_track) {
        const int longest = *std::max_element(d.len, d.len + d.B) + 1;
        blocks += kvc * ((longest + WT_SPAN - 1) / WT_SPAN);
    }
    auto combine = ctx->q4_track ? q4_combine_kernel<true> : q4_combine_kernel<false>;
    lc.gridDim = dim3(blocks, d.B);
    lc.blockDim = dim3(256);
    lc.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&lc, combine, d, (const float*)ctx->part_o, (const float*)ctx->part_ml, q_gate, out,
                           (const Q4Slot*)L.d_q4, (const float*)ctx->q4_sc);
    if (e != cudaSuccess) return e;
    *n_launch += 3;
    return cudaGetLastError();
}

}  // namespace dz
