// The 8-bit form of Adam's moments.
//
// 256 consecutive elements of a tensor (GS_MOMENT_BLOCK) share one exponent byte
// per moment: e, the float32 exponent field of the largest rounded magnitude.
// m: a sign, 4 exponent bits and 3 mantissa bits; v: 5 exponent bits and 3
// mantissa bits.  An exponent field f >= 1 (top field T = 15 for m, 31 for v)
// over mantissa bits q stands for 2^(e - 127 - T + f) (1 + q / 8), field 0 for
// q times the step of field 1.  The block's scale is a power of two, so the
// grids of different e are nested: a value on the grid stays on it when e moves,
// and a block whose values do not change is written back unchanged.
//
// Rounding adds an offset u in [0, 1) steps and cuts.  To nearest would be wrong
// here: with beta2 = 0.999 a step moves v by about 0.1 %, less than half of any
// 8-bit grid's step, so v would stop moving a few steps after it starts.  u is a
// low-discrepancy sequence over the step count for each element (multiples of
// sqrt(2), begun at the element's index times the golden ratio, modulo 1), so what
// a rounding leaves out comes back after a few steps; it needs no state.
// v's offset is the complement of m's.  A positive v is never rounded to 0, which
// bounds m / sqrt(v): both forms reach about 2^-17 of the block's largest size.
//
// A magnitude is rounded in its float32 bits: bits + u (20 bits) cut to the upper 3
// mantissa bits is floor(x / step + u) * step for every x of a whole binade, and
// its carry moves to the next binade by itself.  Below field 1 the step is fixed:
// x is scaled so that a step is 2^20, cut by adding 2^23 with rounding toward
// zero, and offset in integers.
#pragma once

#include "common.cuh"

namespace gs {

constexpr uint32_t kDitherElement = 0x9E3779B1u;  // odd, close to 2^32 / golden ratio
constexpr uint32_t kDitherStep = 0x6A09E667u;     // fractional bits of sqrt(2)
constexpr int kMomentTopM = 15, kMomentTopV = 31;
// Lowest block exponent: keeps every scale factor below a normal float32.
constexpr uint32_t kMomentMinExp = 64;

// Value of a code's magnitude (exponent field over 3 bits, at bit 20).
template <int kTop>
__device__ __forceinline__ float moment_value(uint32_t field_bits, float block_scale) {
    // as float32 bits the code is an exponent field and mantissa (field 0: a denormal)
    const float one_binade = __uint_as_float((uint32_t)(254 - kTop) << 23);  // 2^(127 - T)
    return __uint_as_float(field_bits) * one_binade * block_scale;
}

// Eight codes (two words) to values; ``e`` the block's exponent byte.
__device__ __forceinline__ void decode_m8(uint2 c, uint32_t e, float (&x)[8]) {
    const float s = __uint_as_float(e << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t w = k < 4 ? c.x : c.y;
        const int b = 8 * (k & 3);
        const uint32_t f = (b < 24 ? w << (20 - b) : w >> 4) & 0x07f00000u;
        const float v = moment_value<kMomentTopM>(f, s);
        x[k] = __uint_as_float(__float_as_uint(v) ^ ((w << (24 - b)) & 0x80000000u));
    }
}

__device__ __forceinline__ void decode_v8(uint2 c, uint32_t e, float (&x)[8]) {
    const float s = __uint_as_float(e << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t w = k < 4 ? c.x : c.y;
        const int b = 8 * (k & 3);
        const uint32_t f = (b < 24 ? w << (20 - b) : w >> 4) & 0x0ff00000u;
        x[k] = moment_value<kMomentTopV>(f, s);
    }
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Codes of the eight magnitudes ``a`` (float32 bits without sign) of this lane's
// share of a block held by one warp, and the block's exponent byte.  ``w``: the
// dither word of the first element.
template <int kTop, bool kPositive>
__device__ __forceinline__ void encode8(const uint32_t (&a)[8], uint32_t w, uint32_t (&code)[8], uint32_t& e) {
    uint32_t r[8], most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t d = w + (uint32_t)k * kDitherElement;
        r[k] = a[k] + ((kPositive ? ~d : d) >> 12);
        most = max(most, r[k]);
    }
    most = __reduce_max_sync(kFull, most) >> 23;
    e = min(max(most, kMomentMinExp), 255u);
    const uint32_t low = (e - (kTop - 1)) << 23;  // smallest magnitude with exponent field 1
    const uint32_t base = (e - kTop) << 3;
    bool small = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        code[k] = a[k] < low ? 0u : (r[k] >> 20) - base;
        small |= a[k] < low && a[k] != 0;
    }
    if (__any_sync(kFull, small)) {
        // step of field 0 -> 2^20: the factor is 2^(127 + 3 + 20 - (e - (T - 1)))
        const float f = __uint_as_float((277u + (kTop - 1) - e) << 23);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (a[k] < low) {
                const float y = __fadd_rz(__fmul_rn(__uint_as_float(a[k]), f), 8388608.0f);
                const uint32_t d = w + (uint32_t)k * kDitherElement;
                uint32_t c = (__float_as_uint(y) - 0x4B000000u + ((kPositive ? ~d : d) >> 12)) >> 20;
                if (kPositive && c == 0 && a[k] != 0) c = 1;
                if (a[k] == 0) c = 0;
                code[k] = c;
            }
        }
    }
}

// A lane's eight values of both moments -> codes, stored with the block's
// exponents.  All 32 lanes of the warp that holds the block take part.
__device__ __forceinline__ void store_moments8(const float (&m)[8], const float (&v)[8], uint32_t i, uint32_t step_word,
                                               uint8_t* mc, uint8_t* vc, uint8_t* me, uint8_t* ve) {
    const uint32_t w = i * kDitherElement + step_word;
    uint32_t a[8], c[8], e;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(m[k]) & 0x7fffffffu;
    encode8<kMomentTopM, false>(a, w, c, e);
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = (c[k] & 0x7fu) | ((__float_as_uint(m[k]) >> 24) & 0x80u);
    __stcs(reinterpret_cast<uint2*>(mc), make_uint2(pack_bytes(c[0], c[1], c[2], c[3]),
                                                    pack_bytes(c[4], c[5], c[6], c[7])));
    if ((threadIdx.x & 31) == 0) *me = (uint8_t)e;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(v[k]) & 0x7fffffffu;
    encode8<kMomentTopV, true>(a, w, c, e);
    __stcs(reinterpret_cast<uint2*>(vc), make_uint2(pack_bytes(c[0], c[1], c[2], c[3]),
                                                    pack_bytes(c[4], c[5], c[6], c[7])));
    if ((threadIdx.x & 31) == 0) *ve = (uint8_t)e;
}

}  // namespace gs
