// q4.cuh -- the 4-bit KV cache: row format, tile layout and the device functions
// that write rows into tiles and read them back.
//
// A row is one position of one kv head, K or V: 256 values in 8 groups of 32.
//   t = max|x| / 7 of the group; s = t rounded to 4 significant bits (nearest
//   even, grid 2^-17 below 2^-14), at most 896; code = clamp(rint(x / s), -7, 7);
//   the held value is code * s.  NaN is held as 0, infinities saturate, a group
//   whose s rounds to 0 is held as 0.
// Rounding the scale to the nearest (not up) loses nothing from 2^-14 on: t / s <= 17/16,
// so the largest |x| / s is 7.44 and still lands within half a step of code 7.
// s is a positive f16 whose low 7 bits are zero, so 8 bits of it are stored
// (f16 bits >> 7).  code * s has at most 3 + 4 significant bits: exact in f16, so
// the matrix instructions multiply the held values themselves, with no second
// rounding and no scale in an epilogue.  896 is the largest s for which 72 * s,
// the constant of the unpacking below, is still an f16.
//
// Where a value next to a border falls must not depend on rounding in the arithmetic
// before it, so K's codes are those of a norm and rotation in f64: f32 with a bound on
// its error decides nearly every row, f64 the others.  Given values (V, imported rows)
// are decided exactly in f32.
//
// Tile: 16 positions of one kv head, 4352 bytes (K codes 2048, V codes 2048, K
// scales 128, V scales 128), in the register order of mma.m16n8k16, so that a warp
// reads a tile with 16-byte loads and no shuffles.  With r = lane / 4, c = lane % 4:
//   K codes  [pos / 8][i 0..1][lane (r = pos % 8)][4 words]: word w = 4 i + j holds
//            dims 64 c + 8 w .. + 7 of that position, dim e at bit (e & 1) * 16 + (e >> 1) * 4
//   V codes  [i 0..3][c][(r + 2 c) % 8][4 words]: word m = 4 i + j holds dims 32 r + 2 m (A) and
//            32 r + 2 m + 1 (B) at positions 2c, 2c+1, 2c+8, 2c+9: position 2c + u + 8 w
//            at bit u * 16 + w * 4, dim B 8 bits above dim A.  A position lies in four
//            lines of 128 bytes (its c); the rotation by 2 c keeps a warp's 16-byte loads
//            free of bank conflicts.
//   K scales [lane][4]: (pos r, group 2c), (r, 2c+1), (r + 8, 2c), (r + 8, 2c+1)
//   V scales [lane][4]: group r at positions 2c, 2c+1, 2c+8, 2c+9
// Codes are stored as code + 8.  Unwritten positions hold finite scales always
// (the cache starts zeroed), since a masked probability of 0 still multiplies V.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dz_internal.h"

namespace dz {
namespace q4 {

constexpr float SCALE_MAX = 896.0f;
constexpr uint32_t SCALE_MAX_BYTE = 24u << 3 | 6u;            // 896 = 1.75 * 2^9
constexpr int OFF_V = 2048, OFF_KS = 4096, OFF_VS = 4224;
static_assert(OFF_VS + 128 == Q4_TILE_BYTES, "tile layout");
static_assert(Q4_TILE_BYTES % 16 == 0, "tiles move by bulk copies");

// About a millisecond, for what is in flight after a wait that ran into its limit.
__device__ __forceinline__ void settle() {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// ---- f32 pairs in one operation --------------------------------------------------------
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t a, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// ---- scales ------------------------------------------------------------------------
// s (as stored byte) from the group's largest magnitude: 4 significant bits of amax / 7 by
// f32, then decided exactly.  A border lies half a step from s, at 7 s +- 3.5 steps of
// amax, and amax - 7 s is exact there (the two are within a factor of 2), in F's precision:
// no division, and f64 for f64 values alone.
template <typename F>
__device__ __forceinline__ uint32_t scale_byte(F amax) {
    const float t = fminf((float)amax * (1.0f / 7.0f), SCALE_MAX);
    uint32_t byte;                                             // exponent << 3 | 3 fraction bits, of f16
    if (t < 6.103515625e-05f) {                                // 2^-14: the grid is 2^-17, f16's subnormals
        byte = (uint32_t)__float2int_rn(t * 131072.0f);        // 0..8 (8 = the smallest normal)
    } else {
        const uint32_t b = __float_as_uint(t);
        byte = ((b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20) - ((127 - 15) << 3);
    }
    const float s = __half2float(__ushort_as_half((unsigned short)(byte << 7)));
    const float step = __half2float(__ushort_as_half((unsigned short)((byte + 1) << 7))) - s;
    const bool binade = (byte & 7u) == 0u && byte > 8u;        // the step below is half as long
    const F d = fma((F)-7, (F)s, amax), up = (F)3.5 * (F)step, down = binade ? (F)0.5 * up : up;
    const bool odd = byte & 1u;
    if (d > up || (d == up && odd)) byte += 1;
    else if (d < -down || (d == -down && odd)) byte -= 1;
    return min(byte, SCALE_MAX_BYTE);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}
// code + 8 of x: the nearest whole multiple k s (ties to even) within 7 s, decided exactly.
// inv = 1 / s (0 if s is 0), an approximation.
constexpr float ROUND8 = 12582920.0f;                          // 1.5 * 2^23 + 8: x + this is an integer, x + 8 its low bits
// f64: an approximate k, corrected by the remainder, which is exact where k s and x are within
// a factor of 2, and for k = 0; that leaves |k| = 1 with |x| just below s / 2, where it may be
// rounded to s / 2: the tie goes to 0, as x does.
__device__ __forceinline__ uint32_t code8(double x, float s, float inv) {
    x = fmin(fmax(x, -7.0 * s), 7.0 * s);
    const float t = fmaf((float)x, inv, ROUND8);
    const double d = fma((double)(ROUND8 - t), (double)s, x), h = 0.5 * s;
    const bool odd = __float_as_uint(t) & 1u;
    const float up = d > 0.0 ? 1.0f : -1.0f;
    return __float_as_uint(fabs(d) > h || (odd && fabs(d) == h && s > 0.0f) ? t + up : t) & 15u;
}
// f32: the quotient, corrected to the nearest f32.  x has 24 bits and s 4, so a quotient that is
// no tie lies at least 0.53 units in the last place from one (1 / 1.875), and a tie is an f32.
__device__ __forceinline__ uint32_t code8(float x, float s, float inv) {
    x = fminf(fmaxf(x, -7.0f * s), 7.0f * s);
    const float u = x * inv;
    return __float_as_uint(fmaf(fmaf(-u, s, x), inv, u) + ROUND8) & 15u;
}

// two scale bytes (bits 0..7 and 16..23) -> an f16 pair
__device__ __forceinline__ uint32_t scale_pair(uint32_t bytes) { return bytes << 7; }

// ---- unpacking ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// (x & mask) | magic in one operation (written in C++ it becomes two: one immediate each)
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(magic));
    return d;
}
constexpr uint32_t NEG72 = 0xD480D480u;                        // f16 pair of -72
// Nibbles n at bits 4..7 and 20..23 of x -> the f16 pair (n - 8) * s.  Under the
// exponent of 64 those bits have weights 8, 4, 2, 1: 64 + n.  (64 + n) s - 72 s in
// one fused operation is exact; c = -72 s.
__device__ __forceinline__ uint32_t unpack(uint32_t x, uint32_t s, uint32_t c) {
    return hfma2_u(and_or(x, 0x00F000F0u, 0x54005400u), s, c);
}

// The matrix loops unpack a word's four pairs from w and w >> 8 alone: nibbles at bits
// 0..3 and 16..19 under the exponent of 1024 (weights 8 4 2 1: 1024 + n), nibbles at bits
// 4..7 and 20..23 under that of 64.  -1032 s would leave f16 at s = 64, so these work with
// s / 16 and give value / 16, still exact (s / 16 is a multiple of 2^-21, f16's grid 2^-24).
struct Scale16 { uint32_t s, c_lo, c_hi; };                    // f16 pairs: s / 16, -1032 s / 16, -72 s / 16
__device__ __forceinline__ Scale16 scale16(uint32_t pair) {    // pair: scale_pair()
    return {hmul2_u(pair, 0x2C002C00u), hmul2_u(pair, 0xD408D408u), hmul2_u(pair, 0xC480C480u)};
}
__device__ __forceinline__ uint32_t unpack_lo(uint32_t x, const Scale16& k) {
    return hfma2_u(and_or(x, 0x000F000Fu, 0x64006400u), k.s, k.c_lo);
}
__device__ __forceinline__ uint32_t unpack_hi(uint32_t x, const Scale16& k) {
    return hfma2_u(and_or(x, 0x00F000F0u, 0x54005400u), k.s, k.c_hi);
}

// ---- rotary positions ----------------------------------------------------------------
// Angle of pair i at position p in half turns, reduced to [-1, 1]: p * base^(-2i/64) / pi.
// In f64: at p = 10^6 an f32 angle is off by 0.03.
__device__ __forceinline__ double rope_half_turns(int p, double turn) {
    const double u = (double)p * turn;
    return u - 2.0 * rint(0.5 * u);
}
// (cos, sin) of pair i at a token's three positions
__device__ __forceinline__ double2 rope_cs(const RopeAxes& a, int i, int t, int h, int w) {
    const int ax = a.axis[i];
    double s, c;
    sincospi(rope_half_turns(ax == 0 ? t : (ax == 1 ? h : w), a.turn[i]), &s, &c);
    return make_double2(c, s);
}

// ---- a row in registers ----------------------------------------------------------------
// Lane l holds dims 8 l .. 8 l + 7 of a row (a group of 32 = 4 lanes).

// RMS norm, weight and rotation (attention.rs:92-113, with the reference's '+' sign for
// both halves, math/rope.rs:205-210), in f64 for rows that are quantised and in f32 for
// the others.  cs: (cos, sin) of the 32 pairs.  The partner of dim i < 32 is i + 32:
// lane ^ 4.
__device__ __forceinline__ double inv_sqrt(double x) {         // Newton's iteration from f32's: 2^-23, 2^-45, 2^-53
    if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);        // where f32's would lose bits or overflow
    double g = (double)rsqrtf((float)x);
#pragma unroll
    for (int i = 0; i < 2; ++i) g = fma(fma(-x * g, g, 1.0), 0.5 * g, g);
    return g;
}
__device__ __forceinline__ float inv_sqrt(float x) { return 1.0f / sqrtf(x); }
// 1 / rms of a row whose mean square v = sum / 256 + eps left f32, or the range where it keeps its bits: taken of the row
// times a power of two.  (An infinity in the row: 0, as 1 / sqrt has it.)
__device__ __forceinline__ bool out_of_range(float v) { return !(v > 1e-30f && v < 1e38f); }   // the same for the whole warp
__device__ __forceinline__ float scaled_inv_rms(const float (&x)[8], float v, float eps) {
    const float up = v < 1.0f ? 0x1p80f : 0x1p-80f;
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e] * up, x[e] * up, ss);
    return up * inv_sqrt(fmaf(warp_sum(ss), 1.0f / (float)HD, eps * up * up));
}
template <typename F, typename C>
__device__ __forceinline__ void norm_rotate(F (&x)[8], const float* __restrict__ w, const C* cs, float eps, int lane) {
    F ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const F v = ss / (F)HD + (F)eps;
    F inv = inv_sqrt(v);
    if constexpr (sizeof(F) == sizeof(float)) {
        if (out_of_range(v)) inv = scaled_inv_rms(x, v, eps);
    }
    const float4 w0 = reinterpret_cast<const float4*>(w)[2 * lane], w1 = reinterpret_cast<const float4*>(w)[2 * lane + 1];
    const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (F)wv[e];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const F p = __shfl_xor_sync(0xffffffffu, x[e], 4);
        if (lane < 8) {
            const C c = cs[8 * (lane & 3) + e];
            x[e] = x[e] * (F)c.x + p * (F)c.y;
        }
    }
}

// Rows that are not quantised: lane l holds two runs of 4 dims, at split_dim(l, 0) and
// split_dim(l, 1), such that a rotary pair (i, i + 32) lies in one lane (lanes 0..7), and
// neighbouring lanes' runs are neighbours: a store fills whole sectors.
__device__ __forceinline__ int split_dim(int lane, int run) {
    return lane < 8 ? 4 * lane + 32 * run : 32 + 4 * lane + 96 * run;
}
// Weight (w: this lane's 8) and rotation of a row times inv, in f32; cs: (cos, sin) of pairs 4 l .. 4 l + 3 in lanes 0..7.
__device__ __forceinline__ void scale_rotate_split(float (&x)[8], float inv, const float (&w)[8], const float2 (&cs)[4],
                                                   int lane) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (x[e] * inv) * w[e];
    if (lane < 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = x[e], b = x[e + 4];
            x[e] = fmaf(a, cs[e].x, b * cs[e].y);
            x[e + 4] = fmaf(b, cs[e].x, a * cs[e].y);
        }
    }
}
// RMS norm, weight and rotation.  False, the same for the whole warp, where the row's mean square is out of range: the
// caller takes such rows again behind its loop (norm_rotate_far).  A branch to that in here costs registers and keeps
// rows in flight from overlapping: the rotary pass of 32768 bf16 tokens took 193 us instead of 166.
__device__ __forceinline__ bool norm_rotate_split(float (&x)[8], const float (&w)[8], const float2 (&cs)[4], float eps,
                                                  int lane) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    const float v = fmaf(warp_sum(ss), 1.0f / (float)HD, eps), g = rsqrtf(v);
    scale_rotate_split(x, fmaf(fmaf(-v * g, g, 1.0f), 0.5f * g, g), w, cs, lane);   // one Newton step: to the last bit or so
    return !out_of_range(v);
}
__device__ __forceinline__ void norm_rotate_far(float (&x)[8], const float (&w)[8], const float2 (&cs)[4], float eps,
                                                int lane) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    scale_rotate_split(x, scaled_inv_rms(x, fmaf(warp_sum(ss), 1.0f / (float)HD, eps), eps), w, cs, lane);
}
// The (cos, sin) that norm_rotate_split wants, from a lane's own pair (lane = pair).
__device__ __forceinline__ void spread_pairs(float2 own, float2 (&cs)[4], int lane) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cs[e].x = __shfl_sync(0xffffffffu, own.x, (4 * lane + e) & 31);
        cs[e].y = __shfl_sync(0xffffffffu, own.y, (4 * lane + e) & 31);
    }
}
// (cos, sin) of pair i at a token's three positions in f32, the angle reduced in f64
__device__ __forceinline__ float2 rope_cs_f32(const RopeAxes& a, int i, int t, int h, int w) {
    const int ax = a.axis[i];
    float s, c;
    sincospif((float)rope_half_turns(ax == 0 ? t : (ax == 1 ? h : w), a.turn[i]), &s, &c);
    return make_float2(c, s);
}
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ uint2 load4(const __nv_bfloat16* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ float4 as_f32(float4 x) { return x; }
__device__ __forceinline__ float4 as_f32(uint2 u) {
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
}
// A lane's 8 dims of a row as they lie in memory: several rows can be in flight.
template <typename T>
struct SplitRow {
    decltype(load4((const T*)nullptr)) a, b;
    __device__ __forceinline__ void load(const T* row, int lane) {
        a = load4(row + split_dim(lane, 0));
        b = load4(row + split_dim(lane, 1));
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
        const float4 u = as_f32(a), v = as_f32(b);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    }
};
template <typename T>
__device__ __forceinline__ void load_split(const T* row, int lane, float (&x)[8]) {
    SplitRow<T> r;
    r.load(row, lane);
    r.values(x);
}

// Quantise the row, exactly: the stored scale byte of this lane's group and the 8 codes + 8.
template <typename F>
__device__ __forceinline__ uint32_t quantise(F (&x)[8], uint32_t (&code)[8]) {
    F a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = x[e] == x[e] ? x[e] : (F)0;
        a = fmax(a, fabs(x[e]));
    }
    a = fmax(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = fmax(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const uint32_t sb = scale_byte(a);
    const float s = scale_value(sb);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    inv = s > 0.0f ? inv : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = code8(x[e], s, inv);
    return sb;
}

// The same from f32 values that are off by at most 7e-7 of their own magnitude and of `from`
// (0, or what they were computed from): false where that could change a code or a scale, that
// is where one lies within about 1e-5 of a border, and for NaN.  A row is undecided about once
// in 50 times; f64 for every row took three times as many instructions.
__device__ __forceinline__ bool quantise_f32(const float (&x)[8], float from, uint32_t (&code)[8], uint32_t& sb) {
    float a = 0.0f, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a = fmaxf(a, fabsf(x[e]));
        sum += x[e];
    }
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
    // |error of a value| <= 7e-7 (a + from) <= 3.5e-6 a = 2.5e-5 s where `from` is at most 4 a
    bool ok = sum == sum && from <= 4.0f * a;
    const float t = fminf(a * (1.0f / 7.0f), SCALE_MAX);
    if (t < 6.103515625e-05f) {                                // as in scale_byte
        const float u = t * 131072.0f, r = rintf(u);
        sb = (uint32_t)(int)r;
        ok = ok && fabsf(u - r) < 0.4999f;
    } else {
        const uint32_t b = __float_as_uint(t);
        sb = ((b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20) - ((127 - 15) << 3);
        ok = ok && (b & 0xFFFFFu) - (0x80000u - 128u) > 256u;  // 128 steps of 2^-24..2^-23 from a border
    }
    const float s = scale_value(sb);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    inv = s > 0.0f ? inv : 0.0f;
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float u = fminf(fmaxf(x[e] * inv, -7.0f), 7.0f), r = u + ROUND8;
        code[e] = __float_as_uint(r) & 15u;
        off = fmaxf(off, fabsf(u - (r - ROUND8)));
    }
    return ok && off < 0.5f - 4e-5f;
}
// A row of K: normalised, rotated, quantised as in f64.  csf: its 32 angles (rope_cs_f32), t, h, w:
// the positions they are of; cs: the warp's place for them in f64.
__device__ __forceinline__ uint32_t quantise_key(const float (&x)[8], const float* __restrict__ weight,
                                                 const float2* csf, double2* cs, const RopeAxes& axes, int t, int h, int w,
                                                 float eps, int lane, uint32_t (&code)[8]) {
    uint32_t sb;
    // f32: the norm is off by at most 5e-7 (13 roundings of its sum, halved, and its root), a value by two
    // roundings more, sine and cosine by 3.1e-7 (1.9e-7 of them the angle's rounding)
    float y[8], ss = 0.0f, from = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    const float v = fmaf(warp_sum(ss), 1.0f / (float)HD, eps), g = rsqrtf(v);
    const float inv = fmaf(fmaf(-v * g, g, 1.0f), 0.5f * g, g);
    const float4* wp = reinterpret_cast<const float4*>(weight) + 2 * lane;
    const float4 w0 = wp[0], w1 = wp[1];
    const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        y[e] = (x[e] * inv) * wv[e];
        from = fmaxf(from, fabsf(y[e]));
    }
    from = lane < 8 ? fmaxf(from, __shfl_xor_sync(0xffu, from, 4)) : 0.0f;   // the rotated dims and their partners
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float p = __shfl_xor_sync(0xffffffffu, y[e], 4);
        if (lane < 8) {
            const float2 c = csf[8 * (lane & 3) + e];
            y[e] = fmaf(y[e], c.x, p * c.y);
        }
    }
    bool ok = quantise_f32(y, from, code, sb);
    ok = ok && v > 1e-30f && v < 1e30f;                        // no overflow or lost bits on the way
    if (__any_sync(0xffffffffu, !ok)) {
        cs[lane] = rope_cs(axes, lane, t, h, w);
        __syncwarp();
        double z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = x[e];
        norm_rotate(z, weight, cs, eps, lane);
        sb = quantise(z, code);
    }
    return sb;
}

// Writes K's codes and scale of position p (0..15) of a tile.  Lane l's 8 dims are one
// word: c = l / 8, word l % 8.
__device__ __forceinline__ void put_k(uint8_t* tile, int p, int lane, const uint32_t (&code)[8], uint32_t sb) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code[e] << ((e & 1) * 16 + (e >> 1) * 4);
    const int c = lane >> 3, ws = lane & 7, n = p & 7;
    *reinterpret_cast<uint32_t*>(tile + ((p >> 3) * 2 + (ws >> 2)) * 512 + (n * 4 + c) * 16 + (ws & 3) * 4) = w;
    const int g = lane >> 2;
    if ((lane & 3) == 0) tile[OFF_KS + (n * 4 + (g >> 1)) * 4 + (p >> 3) * 2 + (g & 1)] = (uint8_t)sb;
}
// Byte offset of V's words 4 i .. 4 i + 3 of (r, c).
__device__ __forceinline__ int v_at(int i, int r, int c) { return OFF_V + i * 512 + c * 128 + ((r + 2 * c) & 7) * 16; }
// The four V words of lane l's dims at column c: group r = l / 4, words 4 (l % 4) .. + 3.
__device__ __forceinline__ uint4* v_words(uint8_t* tile, int lane, int c) {
    return reinterpret_cast<uint4*>(tile + v_at(lane & 3, lane >> 2, c));
}
// The same words with position p's nibbles replaced by the codes.
__device__ __forceinline__ void merge_v(uint4& w, int p, const uint32_t (&code)[8]) {
    const int sh = (p & 1) * 16 + (p >> 3) * 4;
    const uint32_t keep = ~(0x0F0Fu << sh);
    w.x = (w.x & keep) | ((code[0] | code[1] << 8) << sh);
    w.y = (w.y & keep) | ((code[2] | code[3] << 8) << sh);
    w.z = (w.z & keep) | ((code[4] | code[5] << 8) << sh);
    w.w = (w.w & keep) | ((code[6] | code[7] << 8) << sh);
}
__device__ __forceinline__ void put_v_scale(uint8_t* tile, int p, int lane, uint32_t sb) {
    if ((lane & 3) == 0)
        tile[OFF_VS + ((lane >> 2) * 4 + ((p & 7) >> 1)) * 4 + (p & 1) + (p >> 3) * 2] = (uint8_t)sb;
}

// V codes of positions [p0, p1) of one tile, from the warps of a block of 512 threads (a word
// holds four positions): gathered in shared memory, then merged into the tile.
struct TileMerge {
    uint32_t code[512];
    // by every thread before the first tile (end() leaves it ready for the next)
    __device__ __forceinline__ void begin() { code[threadIdx.x] = 0u; }
    // position p's codes, by one warp, after a barrier behind begin() or the last end()
    __device__ __forceinline__ void add(int p, int lane, const uint32_t (&c)[8]) {
        const int at = (v_at(lane & 3, lane >> 2, (p & 7) >> 1) - OFF_V) / 4, sh = (p & 1) * 16 + (p >> 3) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) atomicOr(&code[at + i], (c[2 * i] | c[2 * i + 1] << 8) << sh);
    }
    __device__ __forceinline__ void end(uint8_t* tile, int p0, int p1) {
        __syncthreads();
        uint32_t* w = reinterpret_cast<uint32_t*>(tile + OFF_V) + threadIdx.x;
        uint32_t m = 0;                                        // the nibbles of column c's positions 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = 2 * ((threadIdx.x >> 5) & 3) + (k & 1) + 8 * (k >> 1);
            if (p >= p0 && p < p1) m |= 0x0F0Fu << ((p & 1) * 16 + (p >> 3) * 4);
        }
        const uint32_t c = code[threadIdx.x];
        if (m == 0xFFFFFFFFu) *w = c;
        else if (m) *w = (*w & ~m) | c;
        code[threadIdx.x] = 0u;
    }
};

// Reads lane l's 8 dims of K or V at position p of a tile as f16 pairs.
__device__ __forceinline__ void get_k(const uint8_t* tile, int p, int lane, uint32_t (&h)[4]) {
    const int c = lane >> 3, ws = lane & 7, n = p & 7, g = lane >> 2;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + ((p >> 3) * 2 + (ws >> 2)) * 512 + (n * 4 + c) * 16 +
                                                          (ws & 3) * 4);
    const uint32_t b = tile[OFF_KS + (n * 4 + (g >> 1)) * 4 + (p >> 3) * 2 + (g & 1)];
    const uint32_t s = scale_pair(b | b << 16), k = hmul2_u(s, NEG72);
    h[0] = unpack(w << 4, s, k);
    h[1] = unpack(w, s, k);
    h[2] = unpack(w >> 4, s, k);
    h[3] = unpack(w >> 8, s, k);
}
__device__ __forceinline__ void get_v(const uint8_t* tile, int p, int lane, uint32_t (&h)[4]) {
    const int c = (p & 7) >> 1;
    const uint4 w = *reinterpret_cast<const uint4*>(tile + v_at(lane & 3, lane >> 2, c));
    const uint32_t b = tile[OFF_VS + ((lane >> 2) * 4 + c) * 4 + (p & 1) + (p >> 3) * 2];
    const uint32_t s = scale_pair(b | b << 16), k = hmul2_u(s, NEG72);
    const int sh = (p & 1) * 16 + (p >> 3) * 4;
    const uint32_t x[4] = {w.x >> sh, w.y >> sh, w.z >> sh, w.w >> sh};
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = unpack((x[i] & 0xFu) << 4 | (x[i] & 0xF00u) << 12, s, k);
}

// The same for 4 dims, 4 l + 128 half.
__device__ __forceinline__ void get_k4(const uint8_t* tile, int p, int lane, int half, uint32_t (&h)[2]) {
    const int w8 = (lane >> 1) + 16 * half, c = w8 >> 3, ws = w8 & 7, n = p & 7, g = w8 >> 2;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + ((p >> 3) * 2 + (ws >> 2)) * 512 + (n * 4 + c) * 16 +
                                                          (ws & 3) * 4) >> (8 * (lane & 1));
    const uint32_t b = tile[OFF_KS + (n * 4 + (g >> 1)) * 4 + (p >> 3) * 2 + (g & 1)];
    const uint32_t s = scale_pair(b | b << 16), k = hmul2_u(s, NEG72);
    h[0] = unpack(w << 4, s, k);
    h[1] = unpack(w, s, k);
}
__device__ __forceinline__ void get_v4(const uint8_t* tile, int p, int lane, int half, uint32_t (&h)[2]) {
    const int w8 = (lane >> 1) + 16 * half, c = (p & 7) >> 1;
    const uint2 w = *reinterpret_cast<const uint2*>(tile + v_at(w8 & 3, w8 >> 2, c) + 8 * (lane & 1));
    const uint32_t b = tile[OFF_VS + ((w8 >> 2) * 4 + c) * 4 + (p & 1) + (p >> 3) * 2];
    const uint32_t s = scale_pair(b | b << 16), k = hmul2_u(s, NEG72);
    const int sh = (p & 1) * 16 + (p >> 3) * 4;
    const uint32_t x[2] = {w.x >> sh, w.y >> sh};
#pragma unroll
    for (int i = 0; i < 2; ++i) h[i] = unpack((x[i] & 0xFu) << 4 | (x[i] & 0xF00u) << 12, s, k);
}

}  // namespace q4
}  // namespace dz
