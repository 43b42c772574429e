// q4_evict.cu -- eviction from 4-bit KV caches by accumulated attention weight.
//
// Of each kv head of a sequence the last `recent` entries stay, and of the others the
// heaviest, `keep` in all, in their order; equal weights: the earlier entry stays.
//
// One kernel, a cluster of CTAs per (sequence, kv head):
//   1. the weight of the last entry that stays: radix selection over the weights as ordered
//      32-bit keys, 11 + 11 + 10 bits, a histogram per CTA, which every CTA reads from all
//      (distributed shared memory, 16 bytes at a time; adding them up by remote atomics
//      took 45 ns an instruction);
//   2. the indices that stay: each CTA counts its stretch of entries, prefix sums over the
//      cluster, then writes its part of the list in order;
//   3. the rows move, 16 positions a warp at a time: a round of destination tiles is built
//      in shared memory from its sources, and written once every CTA of the cluster has
//      read its own.  An entry only moves towards the front, so the sources of a later
//      round lie behind everything that an earlier one writes: source and destination may
//      be the same sequence.
// Bound by latency (cluster barriers and block scans of the selection, then two dependent
// reads per moved row): one sequence of 4352 to 4096, 25 us; 13 of 9000-32768 to 2048 (63 MB),
// 60 us, half of it the scattered reads (about 900 bytes in pieces of 32 to 128 per kept row).
#include <algorithm>

#include "q4.cuh"

namespace dz {
namespace q4 {

constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32;
constexpr int EV_PER = 8;                        // consecutive entries of a thread
constexpr int EV_BATCH = EV_PER * EV_THREADS;    // entries that a CTA looks at at a time

struct Evict {
    int B, kvc;
    int32_t src[MAXB], dst[MAXB], len[MAXB];
    int32_t keep[MAXB], recent[MAXB];            // entries that stay (<= len), of which the last ones
    int64_t out[MAXB];                           // first index of the sequence in the list
};

struct alignas(16) EvictSmem {
    union {
        struct {                                 // step 3: one tile per warp
            uint8_t tile[EV_WARPS][Q4_TILE_BYTES];
            float wts[EV_WARPS][Q4_TILE];
        };
        struct {                                 // step 1
            uint32_t hist[3][2048];
        };
    };
    uint32_t scan[EV_WARPS], scan2[EV_WARPS];
    uint32_t found[3];                           // bin, entries above it, entries in it
    alignas(8) uint32_t count[2];                // this CTA's entries above the threshold, and at it
};

// Weights in order as unsigned keys; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    const uint32_t b = __float_as_uint(w + 0.0f);
    if (w != w) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 16 or 8 bytes of the same shared-memory place in CTA `rank` of the cluster
__device__ __forceinline__ uint4 peer_16(const uint32_t* p, uint32_t rank) {
    uint32_t a;
    uint4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 peer_8(const uint32_t* p, uint32_t rank) {
    uint32_t a;
    uint2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}

// Exclusive prefix sums of x over the block's threads, and their total.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* warp_sums, uint32_t& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t v = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < EV_WARPS; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    __syncthreads();
    total = all;
    return before + v - x;
}

// A warp builds the tile of 16 entries whose sources are src[0 .. n) (n <= 16; the rest
// becomes zeros) in shared memory, codes, scales and weights.
__device__ __forceinline__ void build_tile(uint8_t* out, float* wts_out, const Q4Slot& slot, int kvh,
                                           const int32_t* src, int n, int lane) {   // src: written by this kernel
    const int32_t mine = lane < n ? src[lane] : -1;            // source of destination position `lane`
    if (lane < Q4_TILE) wts_out[lane] = mine >= 0 ? slot.wts[(size_t)kvh * slot.cap + mine] : 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {                              // K codes: 8 pieces of 16 bytes a position
        const int id = k * 32 + lane, p = id >> 3, i = (id >> 2) & 1, c = id & 3;
        const int32_t s = __shfl_sync(0xffffffffu, mine, p);
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (s >= 0)
            w = *reinterpret_cast<const uint4*>(slot.tile(kvh, s >> 4) + (((s >> 3) & 1) * 2 + i) * 512 +
                                                ((s & 7) * 4 + c) * 16);
        *reinterpret_cast<uint4*>(out + ((p >> 3) * 2 + i) * 512 + ((p & 7) * 4 + c) * 16) = w;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {                              // K scales: two groups at a time
        const int id = k * 32 + lane, p = id >> 2, c = id & 3;
        const int32_t s = __shfl_sync(0xffffffffu, mine, p);
        uint16_t v = 0;
        if (s >= 0)
            v = *reinterpret_cast<const uint16_t*>(slot.tile(kvh, s >> 4) + OFF_KS + ((s & 7) * 4 + c) * 4 +
                                                   ((s >> 3) & 1) * 2);
        *reinterpret_cast<uint16_t*>(out + OFF_KS + ((p & 7) * 4 + c) * 4 + (p >> 3) * 2) = v;
    }
    // V: lane (r, c) has the words of positions 2c, 2c + 1, 2c + 8, 2c + 9
    const int r = lane >> 2, c = lane & 3;
    uint4 w[4] = {};
    uint32_t scales = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int u = q & 1, hi = q >> 1;
        const int32_t s = __shfl_sync(0xffffffffu, mine, 2 * c + u + 8 * hi);
        if (s < 0) continue;
        const uint8_t* tile = slot.tile(kvh, s >> 4);
        const int c_from = (s & 7) >> 1, sh = (s & 1) * 16 + ((s >> 3) & 1) * 4, to = u * 16 + hi * 4;
        scales |= (uint32_t)tile[OFF_VS + (r * 4 + c_from) * 4 + (s & 1) + ((s >> 3) & 1) * 2] << (8 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(tile + v_at(i, r, c_from));
            w[i].x |= ((x.x >> sh) & 0x0F0Fu) << to;
            w[i].y |= ((x.y >> sh) & 0x0F0Fu) << to;
            w[i].z |= ((x.z >> sh) & 0x0F0Fu) << to;
            w[i].w |= ((x.w >> sh) & 0x0F0Fu) << to;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(out + v_at(i, r, c)) = w[i];
    *reinterpret_cast<uint32_t*>(out + OFF_VS + lane * 4) = scales;
}

// EV_CTAS: CTAs of a cluster
template <int EV_CTAS>
__global__ void __launch_bounds__(EV_THREADS, 2)
    q4_evict_kernel(const __grid_constant__ Evict d, const Q4Slot* __restrict__ slots, int32_t* list,
                    int32_t* __restrict__ kept) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    EvictSmem& sm = *reinterpret_cast<EvictSmem*>(smem_raw);
    const int rank = blockIdx.x % EV_CTAS, pair = blockIdx.x / EV_CTAS, b = pair / d.kvc, kvh = pair - b * d.kvc;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Q4Slot src = slots[d.src[b]], dst = slots[d.dst[b]];
    const int n = d.len[b], keep = d.keep[b], recent = d.recent[b];
    const int old = n - recent, need = keep - recent;          // `need` of the first `old` entries stay
    const float* wts = src.wts + (size_t)kvh * src.cap;
    list += d.out[b] * d.kvc + (int64_t)kvh * keep;
    if (kept) kept += d.out[b] * d.kvc + (int64_t)kvh * keep;
    // this CTA's stretch, in batches of EV_BATCH; a stretch of one batch stays in registers
    const int per = (int)(((int64_t)old + EV_CTAS - 1) / EV_CTAS);
    const int lo = (int)min((int64_t)old, (int64_t)rank * per), hi = (int)min((int64_t)old, (int64_t)lo + per);
    const bool select = need > 0 && need < old;                // the same for the whole cluster
    uint32_t key[EV_PER];
    auto load = [&](int at) {
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) {
            const int j = at + EV_PER * tid + i;
            key[i] = j < hi ? weight_key(wts[j]) : 0u;
        }
    };
    const bool one = hi - lo <= EV_BATCH;
    if (select && one) load(lo);

    // ---- 1. threshold: entries with a larger key stay, and the first `ties` with this key
    uint32_t threshold = 0, ties = 0;
    if (select) {
        for (int i = tid; i < 3 * 2048; i += EV_THREADS) (&sm.hist[0][0])[i] = 0;
        __syncthreads();
        uint32_t prefix = 0, left = (uint32_t)need;            // key bits found so far; entries still to find below them
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
            for (int at = lo; at < hi; at += EV_BATCH) {
                if (!one) load(at);
#pragma unroll
                for (int i = 0; i < EV_PER; ++i) {
                    const bool in = at + EV_PER * tid + i < hi &&
                                    (pass == 0 || (key[i] >> (pass == 1 ? 21 : 10)) == prefix);
                    if (in) atomicAdd(&sm.hist[pass][(key[i] >> shift) & (bins - 1)], 1u);
                }
            }
            cluster_sync();
            // this thread's 4 bins, from the highest bin down, over the cluster
            uint32_t c[4] = {};
            const int top = bins - 1 - 4 * tid;
            if (top >= 0) {
                uint4 v[EV_CTAS];
#pragma unroll
                for (int q = 0; q < EV_CTAS; ++q) v[q] = peer_16(&sm.hist[pass][top - 3], q);
#pragma unroll
                for (int q = 0; q < EV_CTAS; ++q) {
                    c[0] += v[q].w;
                    c[1] += v[q].z;
                    c[2] += v[q].y;
                    c[3] += v[q].x;
                }
            }
            uint32_t total, above = block_scan(c[0] + c[1] + c[2] + c[3], sm.scan, total);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < left && left <= above + c[i]) {
                    sm.found[0] = (uint32_t)(top - i);
                    sm.found[1] = above;
                    sm.found[2] = c[i];
                }
                above += c[i];
            }
            __syncthreads();
            prefix = prefix << (pass == 2 ? 10 : 11) | sm.found[0];
            left -= sm.found[1];
            const uint32_t in_bin = sm.found[2];
            __syncthreads();
            // every entry of the bin stays (it often has just one): the key below it is a threshold
            if (pass < 2 && left == in_bin && prefix > 0u) {
                threshold = (prefix << shift) - 1u;
                left = 0;
                break;
            }
            threshold = prefix;
        }
        ties = left;
    }

    // ---- 2. the list of entries that stay
    if (select) {
        uint32_t gt = 0, eq = 0;
        for (int at = lo; at < hi; at += EV_BATCH) {
            if (!one) load(at);
#pragma unroll
            for (int i = 0; i < EV_PER; ++i)
                if (at + EV_PER * tid + i < hi) {
                    gt += key[i] > threshold;
                    eq += key[i] == threshold;
                }
        }
        uint32_t all_gt, all_eq;
        block_scan(gt, sm.scan, all_gt);
        block_scan(eq, sm.scan2, all_eq);
        if (tid == 0) {
            sm.count[0] = all_gt;
            sm.count[1] = all_eq;
        }
        cluster_sync();
        // the CTAs before this one: lane q reads CTA q's counts
        const uint2 theirs = lane < EV_CTAS ? peer_8(sm.count, lane) : make_uint2(0u, 0u);
        const uint32_t gt_before = __reduce_add_sync(0xffffffffu, lane < rank ? theirs.x : 0u);
        uint32_t eq_before = __reduce_add_sync(0xffffffffu, lane < rank ? theirs.y : 0u);
        uint32_t to0 = gt_before + min(eq_before, ties);
        for (int at = lo; at < hi; at += EV_BATCH) {
            if (!one) load(at);
            uint32_t e = 0, stays = 0, at_threshold = 0;       // bit i: entry i
#pragma unroll
            for (int i = 0; i < EV_PER; ++i)
                if (at + EV_PER * tid + i < hi) {
                    stays |= (uint32_t)(key[i] > threshold) << i;
                    at_threshold |= (uint32_t)(key[i] == threshold) << i;
                }
            e = __popc(at_threshold);
            uint32_t batch_eq, eq_at = block_scan(e, sm.scan, batch_eq) + eq_before;
#pragma unroll
            for (int i = 0; i < EV_PER; ++i)
                if (at_threshold >> i & 1u) stays |= (uint32_t)(eq_at++ < ties) << i;
            uint32_t batch, to = block_scan(__popc(stays), sm.scan2, batch) + to0;
#pragma unroll
            for (int i = 0; i < EV_PER; ++i)
                if (stays >> i & 1u) {
                    const int j = at + EV_PER * tid + i;
                    list[to] = j;
                    if (kept) kept[to] = j;
                    ++to;
                }
            eq_before += batch_eq;
            to0 += batch;
        }
    } else if (need > 0) {                                     // nothing leaves
        for (int j = lo + tid; j < hi; j += EV_THREADS) {
            list[j] = j;
            if (kept) kept[j] = j;
        }
    }
    for (int j = rank * EV_THREADS + tid; j < recent; j += EV_CTAS * EV_THREADS) {
        list[need + j] = old + j;
        if (kept) kept[need + j] = old + j;
    }
    cluster_sync();                                            // the list; and no CTA leaves while another reads its words

    // ---- 3. the rows move
    if (d.src[b] == d.dst[b] && keep == n) return;             // nothing leaves: already in place (the whole cluster)
    const int tiles = (keep + Q4_TILE - 1) / Q4_TILE;
    for (int t0 = 0; t0 < tiles; t0 += EV_CTAS * EV_WARPS) {
        const int t = t0 + warp * EV_CTAS + rank;              // few tiles: spread over the CTAs first
        if (t < tiles)
            build_tile(sm.tile[warp], sm.wts[warp], src, kvh, list + (int64_t)t * Q4_TILE,
                       min(Q4_TILE, keep - t * Q4_TILE), lane);
        cluster_sync();                                        // every source of this round has been read
        if (t < tiles) {
            const uint4* from = reinterpret_cast<const uint4*>(sm.tile[warp]);
            uint4* to = reinterpret_cast<uint4*>(dst.tile(kvh, t));
            for (int i = lane; i < Q4_TILE_BYTES / 16; i += 32) to[i] = from[i];
            const int j = t * Q4_TILE + lane;
            if (lane < Q4_TILE && j < keep) dst.wts[(size_t)kvh * dst.cap + j] = sm.wts[warp][lane];
        }
        __syncwarp();                                          // the warp's staging tile is free again
    }
}

}  // namespace q4

cudaError_t q4_evict_setup() {
    cudaError_t e = cudaSuccess;
    for (auto kernel : {q4::q4_evict_kernel<8>, q4::q4_evict_kernel<4>, q4::q4_evict_kernel<2>})
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(q4::EvictSmem));
    return e;
}

template <int CTAS>
static cudaError_t launch_evict(const q4::Evict& d, const Q4Slot* slots, int32_t* list, int32_t* kept, cudaStream_t st) {
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CTAS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(d.B * d.kvc * CTAS);
    lc.blockDim = dim3(q4::EV_THREADS);
    lc.dynamicSmemBytes = sizeof(q4::EvictSmem);
    lc.stream = st;
    lc.attrs = at;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, q4::q4_evict_kernel<CTAS>, d, slots, list, kept);
}

cudaError_t launch_q4_evict(dz_ctx* ctx, int layer, int B, const int32_t* src, const int32_t* dst, const int64_t* keep,
                            const int64_t* recent, int32_t* kept, cudaStream_t st, int* n_launch) {
    const LayerState& L = ctx->layers[layer];
    const int kvc = ctx->cfg.kv_head_count;
    cudaError_t e;
    int64_t rows = 0;
    for (int b = 0; b < B; ++b) rows += std::min<int64_t>(keep[b], L.len[src[b]]);
    if ((e = ensure_q4_scratch(ctx, std::max<int64_t>(rows, 1) * kvc * sizeof(int32_t))) != cudaSuccess) return e;
    int64_t at = 0;
    for (int b0 = 0; b0 < B; b0 += MAXB) {
        q4::Evict d;
        d.B = std::min(MAXB, B - b0);
        d.kvc = kvc;
        for (int b = 0; b < d.B; ++b) {
            const int64_t n = L.len[src[b0 + b]], k = std::min(keep[b0 + b], n);
            d.src[b] = src[b0 + b];
            d.dst[b] = dst[b0 + b];
            d.len[b] = (int32_t)n;
            d.keep[b] = (int32_t)k;
            d.recent[b] = (int32_t)std::min(recent[b0 + b], k);
            d.out[b] = at;
            at += k;
        }
        // as many CTAs per (sequence, kv head) as fit the GPU at once, two per SM (52 pairs of 20000
        // entries: 60 us with 4, 73 with 8, 91 with 2; 4 pairs: 25 us with 8, 35 and 60 with 4 and 2)
        const int pairs = d.B * kvc;
        int32_t* list = static_cast<int32_t*>(ctx->q4_scratch);
        e = pairs * 8 <= 2 * ctx->n_sm   ? launch_evict<8>(d, L.d_q4, list, kept, st)
            : pairs * 4 <= 2 * ctx->n_sm ? launch_evict<4>(d, L.d_q4, list, kept, st)
                                         : launch_evict<2>(d, L.d_q4, list, kept, st);
        if (e != cudaSuccess) return e;
        *n_launch += 1;
    }
    return cudaSuccess;
}

}  // namespace dz
