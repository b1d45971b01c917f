// The 8-bit form of Adam's moments.
//
// 256 consecutive elements of a tensor (GS_MOMENT_BLOCK) share one exponent byte
// per moment: e, the float32 exponent field of the largest rounded magnitude.
// m: a sign, 4 exponent bits and 3 mantissa bits; v: 5 exponent bits and 3
// mantissa bits.  An exponent field f >= 1 (top field T = 15 for m, 31 for v)
// over mantissa bits q stands for 2^(e - 127 - T + f) (1 + q / 8), field 0 for
// q times the step of field 1.  The block's scale is a power of two, so the
// grids of different e are nested: a value on the grid stays on it when e falls,
// and a block whose values do not change is written back unchanged.  When e rises,
// the values below the new field 1 (2^-14 of the block's binade for m, 2^-30 for v)
// are rounded again, to the new step there.
//
// Rounding adds an offset u in [0, 1) steps and cuts.  To nearest would be wrong
// here: with beta2 = 0.999 a step moves v by about 0.1 %, less than half of any
// 8-bit grid's step, so v would stop moving a few steps after it starts.  u is a
// low-discrepancy sequence over the step count for each element (multiples of
// sqrt(2), begun at the element's index times the golden ratio, modulo 1), so what
// a rounding leaves out comes back after a few steps; it needs no state.
// v's offset is the complement of m's.  A positive v is never rounded to 0, which
// bounds m / sqrt(v): both forms reach about 2^-17 of the block's largest size.  The
// price: rounding is without bias down to one step, 2^-33 of the block's binade, and
// below it v is held as that step.  An element whose gradients stay below 2^-16.5
// (1.1e-5) of the block's largest has too large a v and moves less than it should,
// the less the smaller they are; without any gradient its v stays at the step.  A
// value in the last eighth of float32's largest binade may be rounded to infinity.
//
// A magnitude is rounded in its float32 bits: bits + u (20 bits) cut to the upper 3
// mantissa bits is floor(x / step + u) * step for every x of a whole binade, and
// its carry moves to the next binade by itself.  Below L, the smallest value with
// field 1, the step is fixed: L + x, added with rounding toward zero, holds x in
// units of 2^-20 of that step, and its bits less 2^23 continue those of the values
// above.  They are the larger of the two forms exactly where x < L (the bits of a
// float32 are a concave function of it), so one maximum selects, without a branch.
#pragma once

#include "common.cuh"

namespace gs {

constexpr uint32_t kDitherElement = 0x9E3779B1u;  // odd, close to 2^32 / golden ratio
constexpr uint32_t kDitherStep = 0x6A09E667u;     // fractional bits of sqrt(2)
constexpr int kMomentTopM = 15, kMomentTopV = 31;
// Lowest block exponent: keeps every scale factor below a normal float32.
constexpr uint32_t kMomentMinExp = 64;

// A code's value: its bits at bit 20 are an exponent field and mantissa of
// float32 (field 0: a denormal), so one product with 2^(e - T) gives the value.
// For the largest blocks that factor is no float32 and comes in two parts.
template <int kTop>
struct MomentScale {
    float first, second;
    bool two;
    __device__ __forceinline__ explicit MomentScale(uint32_t e) {
        constexpr uint32_t kOne = 254 - kTop;  // field of 2^(127 - T)
        two = e + kOne - 127 > 254;
        first = __uint_as_float((two ? kOne : e + kOne - 127) << 23);
        second = __uint_as_float(e << 23);
    }
};

__device__ __forceinline__ void scale8(float (&x)[8], float f) {
    const float2 ff = make_float2(f, f);
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const float2 y = __fmul2_rn(make_float2(x[k], x[k + 1]), ff);
        x[k] = y.x;
        x[k + 1] = y.y;
    }
}

// Eight codes (two words) to values; ``e`` the block's exponent byte (255: no
// number, or infinity).
__device__ __forceinline__ void decode_m8(uint2 c, uint32_t e, float (&x)[8]) {
    const MomentScale<kMomentTopM> s(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        // sign and magnitude to bits 31 and 26..20: the byte to the top, then an arithmetic shift
        const uint32_t w = (k < 4 ? c.x : c.y) << (24 - 8 * (k & 3));
        x[k] = __uint_as_float((uint32_t)((int32_t)w >> 4) & 0x87f00000u);
    }
    scale8(x, s.first);
    if (s.two) scale8(x, s.second);
}

__device__ __forceinline__ void decode_v8(uint2 c, uint32_t e, float (&x)[8]) {
    const MomentScale<kMomentTopV> s(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t w = k < 4 ? c.x : c.y;
        const int b = 8 * (k & 3);
        x[k] = __uint_as_float((b < 24 ? w << (20 - b) : w >> 4) & 0x0ff00000u);
    }
    scale8(x, s.first);
    if (s.two) scale8(x, s.second);
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The top bytes of four words.
__device__ __forceinline__ uint32_t pack_tops(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// Codes of the eight magnitudes ``a`` (float32 bits without sign) of this lane's
// share of a block held by one warp, and the block's exponent byte.  ``w``: the
// dither word of the first element (v's: the complement, which counts down).
template <int kTop, bool kPositive>
__device__ __forceinline__ void encode8(const uint32_t (&a)[8], uint32_t w, uint32_t (&code)[8], uint32_t& e) {
    constexpr uint32_t kNext = kPositive ? 0u - kDitherElement : kDitherElement;
    uint32_t most = a[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) most = max(most, a[k]);
    most = __reduce_max_sync(kFull, most);
    if ((most >> 20 & 7u) == 7u) {
        // only from the last eighth of a binade can a rounding carry into the next one
#pragma unroll
        for (int k = 0; k < 8; ++k) most = max(most, a[k] + ((w + (uint32_t)k * kNext) >> 12));
        most = __reduce_max_sync(kFull, most);
    }
    e = min(max(most >> 23, kMomentMinExp), 255u);
    const uint32_t low = (e - (kTop - 1)) << 23;  // L, the smallest magnitude with exponent field 1
    const int base = (int)(e - kTop) << 3;
    const float2 low2 = make_float2(__uint_as_float(low), __uint_as_float(low));
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const float2 fixed2 = __fadd2_rz(make_float2(__uint_as_float(a[k]), __uint_as_float(a[k + 1])), low2);
        const float fixed[2] = {fixed2.x, fixed2.y};
#pragma unroll
        for (int j = k; j < k + 2; ++j) {
            const uint32_t z = (uint32_t)max((int)a[j], (int)(__float_as_uint(fixed[j - k]) - (1u << 23)));
            const int c = (int)((z + ((w + (uint32_t)j * kNext) >> 12)) >> 20) - base;
            code[j] = (uint32_t)(kPositive ? max(c, (int)min(a[j], 1u)) : c);
        }
    }
}

// A lane's eight values of both moments -> codes, stored, and the block's
// exponents.  All 32 lanes of the warp that holds the block take part.  kAnyV: v
// may come with a sign (a caller's; the step's own has none).
template <bool kAnyV>
__device__ __forceinline__ void store_moments8(const float (&m)[8], const float (&v)[8], uint32_t i, uint32_t step_word,
                                               uint8_t* mc, uint8_t* vc, uint32_t& me, uint32_t& ve) {
    const uint32_t w = i * kDitherElement + step_word;
    uint32_t a[8], c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(m[k]) & 0x7fffffffu;
    encode8<kMomentTopM, false>(a, w, c, me);
    uint2 out = make_uint2(pack_bytes(c[0], c[1], c[2], c[3]), pack_bytes(c[4], c[5], c[6], c[7]));
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(m[k]);
    out.x = (out.x & 0x7f7f7f7fu) | (pack_tops(a[0], a[1], a[2], a[3]) & 0x80808080u);
    out.y = (out.y & 0x7f7f7f7fu) | (pack_tops(a[4], a[5], a[6], a[7]) & 0x80808080u);
    __stcs(reinterpret_cast<uint2*>(mc), out);
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(v[k]) & (kAnyV ? 0x7fffffffu : 0xffffffffu);
    encode8<kMomentTopV, true>(a, ~w, c, ve);
    __stcs(reinterpret_cast<uint2*>(vc), make_uint2(pack_bytes(c[0], c[1], c[2], c[3]),
                                                    pack_bytes(c[4], c[5], c[6], c[7])));
}

// The exponent bytes of the blocks that a warp meets in up to 32 successive chunks
// of a tensor, one block a chunk: lane l holds those of chunk l.  They are read
// together before the first chunk and written together after the last.  One byte
// read and written per block and chunk, between those of the other warps in the
// same 32-byte sector, made every read wait for its neighbours' writes: a step over
// 59M parameters took 245 us, and 180 us with the bytes moved like this.
constexpr int kSegment = 32;  // the largest group of chunks a block may take

struct BlockExponents {
    uint32_t m, v;
    // ``first``: the warp's block in the segment's first chunk; ``stride``: blocks from chunk to chunk;
    // ``count``: chunks in which the warp has a block
    __device__ __forceinline__ void load(const uint8_t* me, const uint8_t* ve, int64_t first, int stride, int count) {
        const int lane = threadIdx.x & 31;
        m = v = 0;
        if (lane < count) {
            m = me[first + lane * stride];
            v = ve[first + lane * stride];
        }
    }
    __device__ __forceinline__ void store(uint8_t* me, uint8_t* ve, int64_t first, int stride, int count) const {
        const int lane = threadIdx.x & 31;
        if (lane < count) {
            me[first + lane * stride] = (uint8_t)m;
            ve[first + lane * stride] = (uint8_t)v;
        }
    }
    __device__ __forceinline__ void set(int chunk, uint32_t em, uint32_t ev) {
        if ((threadIdx.x & 31) == chunk) {
            m = em;
            v = ev;
        }
    }
};

}  // namespace gs
