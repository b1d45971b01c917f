// AdamW over many tensors in one launch, moments in 32 bits or in 8, and the
// conversions between the two forms.
//
// For element p of a tensor with gradient g, at step t (both counted on the
// device, so a captured step can be replayed; a tensor without a gradient does not
// count the step):
//   g' = c g                       c: grad_scale, times max_norm / norm when clipped
//   m' = b1 m + (1 - b1) g'        v' = b2 v + (1 - b2) g'^2
//   p' = (1 - lr wd) p - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// The moments' operations are rounded to float32 one by one (no fused multiply-
// add), which fixes them bit for bit; all load paths give the same results.  t,
// the bias corrections, the norm and the factors made of them are formed in 64
// bits and rounded once.
//
// A step moves 28 bytes a float32 parameter with 32-bit moments and 16 with 8-bit
// ones.  59M parameters (of measured copy rate, 6.55 TB/s): 256 us (98 %) and 153 us
// (94 %); with 8-bit moments the 52 instructions an element take 59 % of the issue
// slots, so both bounds are near.  Quantizing them takes 97 us (93 %), reading them
// back as bfloat16 56 us (96 %).
#include <float.h>
#include <math.h>

#include "moments8.cuh"
#include "multi_tensor.cuh"

namespace gs {

// Resident blocks per SM and the largest group of chunks a block takes at a time.
// 32-bit moments: the step is a copy of seven streams, and two blocks of 256
// threads already have enough in flight; three are slower, since more reads and
// writes at once disturb one another in DRAM (59M parameters: 256 us with two, 297
// with three), and single chunks keep the blocks closest together (272 us with 16).  8-bit moments:
// nearly as much arithmetic as memory time, so the registers' most, three; groups of
// half the chunks whose exponents a warp can hold (moments8.cuh).
// Where a tensor of the call has rows or odd alignment, its single accesses wait
// longer and one more block per SM is better, which is why such calls have kernels of
// their own.  Columns of a pool of 1M Gaussians, dense gradients: 489 us with three,
// 520 with two; 8-bit moments 421 with four, 449 with three (strided gradients: 636
// and 655; 598 and 629).  Dense float32 parameters at odd addresses: 295 us with three,
// 346 with two; but with 8-bit moments 352 with four and 337 with three, which the
// columns outweigh.
constexpr int kBlocks32 = 2, kBlocks32Rows = 3, kGroup32 = 1;
constexpr int kBlocks8 = 3, kBlocks8Rows = 4, kGroup8 = 16;
constexpr int kBlocksQuantize = 4, kBlocksQuantizeRows = 3;
constexpr int blocks_for(int bits, bool rows) {
    return bits == 32 ? (rows ? kBlocks32Rows : kBlocks32) : (rows ? kBlocks8Rows : kBlocks8);
}
static_assert(kGroup8 <= kSegment, "a warp holds the exponents of a group");

struct AdamWArgs {
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    float* master;
    int64_t* ctl;           // [0] steps taken, [1] blocks that have read it; upper half: whether any tensor missed one
    int64_t* missed;        // steps that passed without a tensor's gradient, by place in the table (null: none ever)
    const float* lr_dev;    // overrides lr
    const double* partials;
    float* norm_out;
    int64_t num_partials;
    double lr, log2_b1, log2_b2, grad_scale, max_norm;
    float b1, b2, omb1, omb2, eps;
    int advance;            // the step's last launch counts the step
};

struct AdamWShared {
    int64_t t;
    double lr, inv_bc1;
    float gscale, inv_sqrt_bc2;
    uint32_t step_word;
    int skip, any_missed;
};

// The bias corrections of a tensor's t-th step (beta^t = 2^(t log2 beta), in 64 bits).
__device__ __forceinline__ double inverse_correction1(double log2_b1, int64_t t) {
    return 1.0 / (1.0 - exp2((double)t * log2_b1));
}
__device__ __forceinline__ float inverse_sqrt_correction2(double log2_b2, int64_t t) {
    return (float)(1.0 / sqrt(1.0 - exp2((double)t * log2_b2)));
}
// Called for the further tensors of a block where any missed a step.  In line, this code between the chunks costs
// every step: a tiny scene in a graph takes 3.6 us instead of 3.4.
__device__ __noinline__ double further_correction1(double log2_b1, int64_t t) {
    return inverse_correction1(log2_b1, t);
}
__device__ __noinline__ float further_correction2(double log2_b2, int64_t t) {
    return inverse_sqrt_correction2(log2_b2, t);
}

// Which of its steps a tensor takes in the optimizer's t-th.
__device__ __forceinline__ int64_t own_step(int64_t t, int64_t missed) { return max(t - missed, (int64_t)1); }

// The gradients' norm; a step for which it is not finite in float32 is skipped.
__device__ __forceinline__ double scaled_norm(const AdamWArgs& a, double sum_of_squares) {
    return fabs(a.grad_scale) * sqrt(sum_of_squares);
}

// What every element of the step shares.  Each block sums the norm's partials
// itself (a few hundred doubles in a fixed order), which needs no launch
// between the norm and the step; the bias corrections of the block's first tensor,
// at ``place``, are formed by other warps meanwhile.
__device__ __forceinline__ void adamw_prologue(const AdamWArgs& a, AdamWShared& sh, int place) {
    int64_t taken, own;
    asm volatile("ld.volatile.global.v2.s64 {%0, %1}, [%2];" : "=l"(taken), "=l"(own) : "l"(a.ctl) : "memory");
    const int64_t missed = a.missed ? a.missed[place] : 0;
    const int64_t t = taken + 1;
    if (threadIdx.x == 32)
        sh.inv_bc1 = inverse_correction1(a.log2_b1, own_step(t, missed));
    else if (threadIdx.x == 64)
        sh.inv_sqrt_bc2 = inverse_sqrt_correction2(a.log2_b2, own_step(t, missed));
    double sq = 0.0;
    if (a.partials) sq = sum_partials(a.partials, a.num_partials);
    if (threadIdx.x == 0) {
        double scale = a.grad_scale;
        bool skip = false;
        if (a.partials) {
            const double norm = scaled_norm(a, sq);
            skip = !isfinite((float)norm);
            if (norm > a.max_norm) scale *= a.max_norm / norm;
            if (blockIdx.x == 0 && a.norm_out) *a.norm_out = (float)norm;
        }
        sh.t = t;
        sh.skip = skip;
        sh.any_missed = a.missed && own >> 32 != 0;
        sh.gscale = (float)scale;
        sh.lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
        sh.step_word = (uint32_t)t * kDitherStep;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        // the last block whose threads have read the count writes the new one; a skipped step is not counted
        __threadfence();
        unsigned int* ticket = reinterpret_cast<unsigned int*>(a.ctl + 1);
        if (atomicAdd(ticket, 1u) == gridDim.x - 1) {
            *ticket = 0;
            if (a.advance && !sh.skip) a.ctl[0] = t;
        }
    }
}

// The parameter, with the hardware's approximate square root and reciprocal: 2
// ulp each on the step, far below the rounding of the parameter it moves.  The
// rounded forms take a slow path where m or v is a denormal, which is where the
// moments of long unseen Gaussians end (0.9^800 of a gradient): a step over a
// scene half of which is unseen took twice as long with them (561 us against 269).
__device__ __forceinline__ float param_update(float p, float m, float v, float inv_sqrt_bc2, float step, float keep,
                                              float eps) {
    float root, inv;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
    const float denom = fmaf(root, inv_sqrt_bc2, eps);  // eps is a normal number, so denom is
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(denom));
    return fmaf(-step, m * inv, p * keep);
}

// What a tensor's elements share in the step.
struct AdamWTensor {
    float step, keep, gscale, inv_sqrt_bc2;
    uint32_t step_word;
};

__device__ __forceinline__ void update8(float (&p)[8], const float (&g)[8], float (&m)[8], float (&v)[8],
                                        const AdamWTensor& t, const AdamWArgs& a) {
    const float2 b1 = make_float2(a.b1, a.b1), omb1 = make_float2(a.omb1, a.omb1);
    const float2 b2 = make_float2(a.b2, a.b2), omb2 = make_float2(a.omb2, a.omb2);
    const float2 c = make_float2(t.gscale, t.gscale);
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        // The moments, every operation rounded by itself: the products of two elements in one instruction, the sums
        // in single ones, because packed products and sums are joined into fused ones even where both name their
        // rounding.
        const float2 gk = __fmul2_rn(make_float2(g[k], g[k + 1]), c);
        const float2 ma = __fmul2_rn(b1, make_float2(m[k], m[k + 1])), mb = __fmul2_rn(omb1, gk);
        const float2 va = __fmul2_rn(b2, make_float2(v[k], v[k + 1])), vb = __fmul2_rn(omb2, __fmul2_rn(gk, gk));
        m[k] = __fadd_rn(ma.x, mb.x);
        m[k + 1] = __fadd_rn(ma.y, mb.y);
        v[k] = __fadd_rn(va.x, vb.x);
        v[k + 1] = __fadd_rn(va.y, vb.y);
        p[k] = param_update(p[k], m[k], v[k], t.inv_sqrt_bc2, t.step, t.keep, a.eps);
        p[k + 1] = param_update(p[k + 1], m[k + 1], v[k + 1], t.inv_sqrt_bc2, t.step, t.keep, a.eps);
    }
}

// ``count`` whole chunks of a tensor from element i on, all accesses 16 bytes wide.
// kWideP: float32 parameters (or masters: kMaster, with 16-bit parameters written
// from them); kWideG: float32 gradients.
template <int kBits, bool kWideP, bool kWideG, bool kMaster>
__device__ __forceinline__ void adamw_chunks(const TensorEntry& e, const AdamWArgs& a, const AdamWTensor& t, int64_t i,
                                             int count, BlockExponents& x) {
    constexpr int kState = kBits / 8;
    const int64_t s = e.state + i;
    char* m_at = static_cast<char*>(a.m) + s * kState;
    char* v_at = static_cast<char*>(a.v) + s * kState;
    const char* g_at = static_cast<const char*>(e.grad) + i * (kWideG ? 4 : 2);
    char* p_at = kMaster ? reinterpret_cast<char*>(a.master + s) : static_cast<char*>(e.param) + i * (kWideP ? 4 : 2);
    char* p16_at = static_cast<char*>(e.param) + i * 2;
    const int p_type = e.param_type, g_type = e.grad_type;
    uint32_t index = (uint32_t)i;
    for (int j = 0; j < count; ++j) {
        Raw8 rm, rv;
        uint2 cm, cv;
        if (kBits == 32) {
            rm = load_raw8<true>(m_at);
            rv = load_raw8<true>(v_at);
        } else {
            cm = __ldcs(reinterpret_cast<const uint2*>(m_at));
            cv = __ldcs(reinterpret_cast<const uint2*>(v_at));
        }
        const Raw8 rg = load_raw8<kWideG>(g_at);
        const Raw8 rp = load_raw8<kWideP || kMaster>(p_at);
        float p[8], g[8], m[8], v[8];
        unpack8<kWideG>(rg, g_type, g);
        if (kBits == 32) {
            unpack8<true>(rm, GS_F32, m);
            unpack8<true>(rv, GS_F32, v);
        } else {
            decode_m8(cm, __shfl_sync(kFull, x.m, j), m);
            decode_v8(cv, __shfl_sync(kFull, x.v, j), v);
        }
        unpack8<kWideP || kMaster>(rp, p_type, p);
        update8(p, g, m, v, t, a);
        store_vec8<kWideP || kMaster, true>(p_at, p_type, p);
        if (kMaster) store_vec8<false, true>(p16_at, p_type, p);
        if (kBits == 32) {
            store_vec8<true, true>(m_at, GS_F32, m);
            store_vec8<true, true>(v_at, GS_F32, v);
        } else {
            uint32_t em, ev;
            store_moments8<false>(m, v, index, t.step_word, reinterpret_cast<uint8_t*>(m_at),
                                  reinterpret_cast<uint8_t*>(v_at), em, ev);
            x.set(j, em, ev);
        }
        m_at += kChunk * kState;
        v_at += kChunk * kState;
        g_at += kChunk * (kWideG ? 4 : 2);
        p_at += kChunk * (kWideP || kMaster ? 4 : 2);
        p16_at += kChunk * 2;
        index += kChunk;
    }
}

// One warp's block of a chunk, where the tensor's end, strides or alignment ask for
// single accesses.  ``em``, ``ev``: the block's exponents; returns the new ones, v's
// in the second byte.  kRows: rows or odd alignment may occur.
template <int kBits, bool kRows>
__device__ __forceinline__ uint32_t adamw_ragged(const TensorEntry& e, const AdamWArgs& a, const AdamWTensor& t,
                                                 int64_t i, uint32_t em, uint32_t ev) {
    const int64_t s = e.state + i;
    const bool masters = a.master != nullptr && e.param_type != GS_F32;
    float p[8], g[8], m[8], v[8];
    if (kRows && !e.grad_vec && !e.param_vec && !masters) {
        float yg[8], yp[8];
        start_rows8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, yg);
        start_rows8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, yp);
        finish_rows8(yg, g);
        finish_rows8(yp, p);
    } else {
        if (kRows)
            load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, e.grad_vec, g);
        else
            load_tail8(e.grad, i, e.n, e.grad_type, g);
        if (masters)
            unpack8(load_raw8(a.master, s, GS_F32), GS_F32, p);
        else if (kRows)
            load_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, e.param_vec, p);
        else
            load_tail8(e.param, i, e.n, e.param_type, p);
    }
    if (kBits == 32) {
        unpack8(load_raw8(a.m, s, GS_F32), GS_F32, m);
        unpack8(load_raw8(a.v, s, GS_F32), GS_F32, v);
    } else {
        decode_m8(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + s), em, m);
        decode_v8(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + s), ev, v);
    }
    update8(p, g, m, v, t, a);
    if (masters) store_vec8(a.master, s, GS_F32, p);
    if (kRows)
        store_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, e.param_vec, p);
    else
        store_tail8(e.param, i, e.n, e.param_type, p);
    if (kBits == 32) {
        store_vec8(a.m, s, GS_F32, m);
        store_vec8(a.v, s, GS_F32, v);
        return 0;
    }
    store_moments8<false>(m, v, (uint32_t)i, t.step_word, static_cast<uint8_t*>(a.m) + s,
                          static_cast<uint8_t*>(a.v) + s, em, ev);
    return em | ev << 8;
}

template <int kBits, int kCap, bool kRows>
__global__ void __launch_bounds__(kMultiThreads, blocks_for(kBits, kRows)) adamw_kernel(
    const __grid_constant__ TensorTable<kCap> tab, const __grid_constant__ AdamWArgs a) {
    __shared__ AdamWShared sh;
    pdl_wait();
    Segments<kCap> seg(tab);
    int chunks;
    int64_t i;
    seg.next(chunks, i);  // every block has a chunk
    int mine, whole;
    int64_t block;
    BlockExponents x;
    // a segment's start: its exponents, in the first segment on their way during the prologue
    auto enter = [&]() {
        const TensorEntry& e = tab.e[seg.tensor];
        i += threadIdx.x * kPerThread;
        warp_chunks(e.n, i, chunks, mine, whole);
        block = (e.state + i) / GS_MOMENT_BLOCK;
        if (kBits == 8) x.load(a.m_exp, a.v_exp, block, kChunk / GS_MOMENT_BLOCK, mine);
    };
    enter();
    adamw_prologue(a, sh, tab.e[seg.tensor].place);
    if (sh.skip) return;
    AdamWTensor t;
    t.gscale = sh.gscale;
    t.step_word = sh.step_word;
    t.inv_sqrt_bc2 = sh.inv_sqrt_bc2;
    double inv_bc1 = sh.inv_bc1;
    for (;;) {
        const TensorEntry& e = tab.e[seg.tensor];
        const double lr = sh.lr * e.lr_scale;
        t.step = (float)(lr * inv_bc1);
        t.keep = (float)(1.0 - lr * e.decay);
        const bool masters = a.master != nullptr && e.param_type != GS_F32;
        int done = 0;
        if (!kRows || (e.param_vec && e.grad_vec)) {
            done = whole;
            const bool wide_g = e.grad_type == GS_F32;
            if (e.param_type == GS_F32) {
                if (wide_g)
                    adamw_chunks<kBits, true, true, false>(e, a, t, i, done, x);
                else
                    adamw_chunks<kBits, true, false, false>(e, a, t, i, done, x);
            } else if (masters) {
                if (wide_g)
                    adamw_chunks<kBits, false, true, true>(e, a, t, i, done, x);
                else
                    adamw_chunks<kBits, false, false, true>(e, a, t, i, done, x);
            } else {
                if (wide_g)
                    adamw_chunks<kBits, false, true, false>(e, a, t, i, done, x);
                else
                    adamw_chunks<kBits, false, false, false>(e, a, t, i, done, x);
            }
        }
        for (; done < mine; ++done) {
            const uint32_t em = kBits == 8 ? __shfl_sync(kFull, x.m, done) : 0;
            const uint32_t ev = kBits == 8 ? __shfl_sync(kFull, x.v, done) : 0;
            const uint32_t both = adamw_ragged<kBits, kRows>(e, a, t, i + (int64_t)done * kChunk, em, ev);
            if (kBits == 8) x.set(done, both & 255u, both >> 8);
        }
        if (kBits == 8) x.store(a.m_exp, a.v_exp, block, kChunk / GS_MOMENT_BLOCK, mine);
        const int before = seg.tensor;
        if (!seg.next(chunks, i)) break;
        // Another tensor's own corrections, where any missed a step.  (At the loop's end: a branch in front of the
        // first chunk's loads costs as much.)
        if (sh.any_missed && seg.tensor != before) {
            const int64_t own = own_step(sh.t, a.missed[tab.e[seg.tensor].place]);
            inv_bc1 = further_correction1(a.log2_b1, own);
            t.inv_sqrt_bc2 = further_correction2(a.log2_b2, own);
        }
        enter();
    }
}

// The tensors of a call that have no gradient, by place from a.missed on.  One block
// counts their missed step, in a launch of its own that only calls with such tensors
// make (4 KB of parameters).
constexpr int kMissedList = 1000;
struct MissedTensors {
    int32_t place[kMissedList];
    int32_t count;
};

__global__ void __launch_bounds__(kMultiThreads) adamw_missed_kernel(const __grid_constant__ MissedTensors list,
                                                                     const __grid_constant__ AdamWArgs a) {
    pdl_wait();
    if (a.partials && !isfinite((float)scaled_norm(a, sum_partials(a.partials, a.num_partials)))) return;
    for (int k = threadIdx.x; k < list.count; k += kMultiThreads) ++a.missed[list.place[k]];
    if (threadIdx.x == 0) reinterpret_cast<uint32_t*>(a.ctl)[3] = 1;
}

// Whole chunks of float32 moments.
__device__ __forceinline__ void quantize_chunks(const TensorEntry& e, uint8_t* mc, uint8_t* vc, int64_t i, int count,
                                                uint32_t step_word, BlockExponents& x) {
    const float* m_at = static_cast<const float*>(e.param) + i;
    const float* v_at = static_cast<const float*>(e.grad) + i;
    mc += e.state + i;
    vc += e.state + i;
    uint32_t index = (uint32_t)i;
    for (int j = 0; j < count; ++j) {
        const Raw8 rm = load_raw8<true>(m_at), rv = load_raw8<true>(v_at);
        float m[8], v[8];
        unpack8<true>(rm, GS_F32, m);
        unpack8<true>(rv, GS_F32, v);
        uint32_t em, ev;
        store_moments8<true>(m, v, index, step_word, mc, vc, em, ev);
        x.set(j, em, ev);
        m_at += kChunk;
        v_at += kChunk;
        mc += kChunk;
        vc += kChunk;
        index += kChunk;
    }
}

template <bool kRows>
__device__ __forceinline__ uint32_t quantize_ragged(const TensorEntry& e, uint8_t* mc, uint8_t* vc, int64_t i,
                                                    uint32_t step_word) {
    float m[8], v[8];
    if (kRows) {
        load_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, e.param_vec, m);
        load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, e.grad_vec, v);
    } else {
        load_tail8(e.param, i, e.n, e.param_type, m);
        load_tail8(e.grad, i, e.n, e.grad_type, v);
    }
    uint32_t em, ev;
    store_moments8<true>(m, v, (uint32_t)i, step_word, mc + e.state + i, vc + e.state + i, em, ev);
    return em | ev << 8;
}

// m (the entries' param) and v (their grad) of any type -> the 8-bit form, with
// step t's offsets.
template <int kCap, bool kRows>
__global__ void __launch_bounds__(kMultiThreads, kRows ? kBlocksQuantizeRows : kBlocksQuantize) moments8_quantize_kernel(
    const __grid_constant__ TensorTable<kCap> tab, uint8_t* mc, uint8_t* vc, uint8_t* me, uint8_t* ve,
    uint32_t step_word) {
    pdl_wait();
    Segments<kCap> seg(tab);
    int chunks;
    int64_t i;
    while (seg.next(chunks, i)) {
        const TensorEntry& e = tab.e[seg.tensor];
        i += threadIdx.x * kPerThread;
        int mine, whole;
        warp_chunks(e.n, i, chunks, mine, whole);
        const int64_t block = (e.state + i) / GS_MOMENT_BLOCK;
        BlockExponents x;
        int done = 0;
        if ((!kRows || (e.param_vec && e.grad_vec)) && e.param_type == GS_F32 && e.grad_type == GS_F32) {
            quantize_chunks(e, mc, vc, i, whole, step_word, x);
            done = whole;
        }
        for (; done < mine; ++done) {
            const uint32_t both = quantize_ragged<kRows>(e, mc, vc, i + (int64_t)done * kChunk, step_word);
            x.set(done, both & 255u, both >> 8);
        }
        x.store(me, ve, block, kChunk / GS_MOMENT_BLOCK, mine);
    }
}

// Whole slabs of codes -> values; a warp a block of 256.
template <int kType>
__global__ void __launch_bounds__(kMultiThreads) moments8_dequantize_kernel(const uint8_t* __restrict__ mc,
                                                                            const uint8_t* __restrict__ vc,
                                                                            const uint8_t* __restrict__ me,
                                                                            const uint8_t* __restrict__ ve, int64_t n,
                                                                            void* m_out, void* v_out) {
    pdl_wait();
    const int64_t i = ((int64_t)blockIdx.x * kMultiThreads + threadIdx.x) * kPerThread;
    if (i >= n) return;
    float x[8];
    const uint2 cm = __ldcs(reinterpret_cast<const uint2*>(mc + i));
    const uint2 cv = __ldcs(reinterpret_cast<const uint2*>(vc + i));
    const uint32_t em = me[i / GS_MOMENT_BLOCK], ev = ve[i / GS_MOMENT_BLOCK];
    decode_m8(cm, em, x);
    store_vec8(m_out, i, kType, x);
    decode_v8(cv, ev, x);
    store_vec8(v_out, i, kType, x);
}

template <int kBits, int kCap>
static const void* adamw_kernel_for(bool all_vec) {
    return all_vec ? (const void*)adamw_kernel<kBits, kCap, false> : (const void*)adamw_kernel<kBits, kCap, true>;
}

template <int kCap>
static int adamw_launches(const gs_tensor* t, int64_t count, int64_t left, int bits, AdamWArgs a,
                          cudaStream_t stream) {
    TensorTable<kCap> tab;
    int64_t* const missed = a.missed;
    for (int64_t at = 0; left > 0;) {
        while (passed_over(t[at])) ++at;
        if (missed) a.missed = missed + at;
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        a.advance = left == 0;
        void* args[] = {&tab, &a};
        const void* k = bits == 32 ? adamw_kernel_for<32, kCap>(tab.all_vec) : adamw_kernel_for<8, kCap>(tab.all_vec);
        const int grid = table_grid(tab, blocks_for(bits, !tab.all_vec), bits == 32 ? kGroup32 : kGroup8);
        GS_TRY(launch_table("adamw_kernel", k, grid, stream, args));
    }
    return GS_OK;
}

static int missed_launches(const gs_tensor* t, int64_t count, AdamWArgs a, cudaStream_t stream) {
    MissedTensors list;
    int64_t* const missed = a.missed;
    for (int64_t at = 0; at < count;) {
        const int64_t from = at;
        list.count = 0;
        for (; at < count && list.count < kMissedList && at - from <= 0x7fffffff; ++at)
            if (t[at].n > 0 && !t[at].grad) list.place[list.count++] = (int32_t)(at - from);
        if (list.count == 0) continue;
        a.missed = missed + from;
        void* args[] = {&list, &a};
        GS_TRY(launch_table("adamw_missed_kernel", (const void*)adamw_missed_kernel, 1, stream, args));
    }
    return GS_OK;
}

template <int kCap>
static int quantize_launches(const gs_tensor* t, int64_t count, int64_t left, uint8_t* m, uint8_t* v, uint8_t* me,
                             uint8_t* ve, uint32_t step_word, cudaStream_t stream) {
    TensorTable<kCap> tab;
    for (int64_t at = 0; left > 0;) {
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        void* args[] = {&tab, &m, &v, &me, &ve, &step_word};
        const void* k = tab.all_vec ? (const void*)moments8_quantize_kernel<kCap, false>
                                    : (const void*)moments8_quantize_kernel<kCap, true>;
        const int blocks = tab.all_vec ? kBlocksQuantize : kBlocksQuantizeRows;
        GS_TRY(launch_table("moments8_quantize_kernel", k, table_grid(tab, blocks, kGroup8), stream, args));
    }
    return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" int gs_adamw_step(const gs_tensor* tensors, int64_t count, const gs_adamw_state* state,
                             const gs_adamw_settings* set, gs_stream_t stream) {
    GS_REQUIRE(state && set, "adamw: null state or settings");
    GS_REQUIRE(state->bits == 32 || state->bits == 8, "adamw: moments have 32 or 8 bits, not %d", state->bits);
    GS_REQUIRE(set->beta1 >= 0.0 && set->beta1 < 1.0 && set->beta2 >= 0.0 && set->beta2 < 1.0,
               "adamw: betas must be in [0, 1)");
    GS_REQUIRE(set->eps >= FLT_MIN && isfinite(set->eps), "adamw: eps must be positive (a normal float32)");
    GS_REQUIRE(isfinite((float)set->grad_scale), "adamw: grad_scale must be finite in float32");
    GS_REQUIRE(set->lr_device || isfinite(set->lr), "adamw: lr must be finite");
    GS_REQUIRE(!set->norm_partials || (set->num_partials >= 0 && set->max_norm > 0.0),
               "adamw: clipping needs a partial count and a positive max_norm");
    GS_REQUIRE(state->counted == 0 || state->counted == 1, "adamw: counted is 0 or 1, not %d", state->counted);
    int64_t live;
    GS_TRY(check_tensors("adamw", tensors, count, kNeedParam | kNeedGrad | (state->counted ? kMayMiss : 0), live));
    if (live == 0) return GS_OK;
    GS_REQUIRE(state->m && state->v && state->control, "adamw: null state pointer");
    GS_REQUIRE(state->bits == 32 || (state->m_exp && state->v_exp), "adamw: 8-bit moments need their exponents");
    GS_REQUIRE(aligned16(state->m) && aligned16(state->v) && aligned16(state->master) && aligned16(state->control),
               "adamw: the state's buffers must be 16-byte aligned");
    AdamWArgs a;
    a.m = state->m;
    a.v = state->v;
    a.m_exp = state->m_exp;
    a.v_exp = state->v_exp;
    a.master = state->master;
    a.ctl = state->control;
    a.missed = state->counted ? state->control + 2 : nullptr;
    a.lr_dev = set->lr_device;
    a.partials = set->norm_partials;
    a.norm_out = set->norm_out;
    a.num_partials = set->num_partials;
    a.lr = set->lr;
    a.log2_b1 = log2(set->beta1);
    a.log2_b2 = log2(set->beta2);
    a.grad_scale = set->grad_scale;
    a.max_norm = set->max_norm;
    a.b1 = (float)set->beta1;
    a.b2 = (float)set->beta2;
    a.omb1 = (float)(1.0 - set->beta1);
    a.omb2 = (float)(1.0 - set->beta2);
    a.eps = set->eps;
    const cudaStream_t st = (cudaStream_t)stream;
    GS_TRY(count <= kSmallTable ? adamw_launches<kSmallTable>(tensors, count, live, state->bits, a, st)
                                : adamw_launches<kLargeTable>(tensors, count, live, state->bits, a, st));
    return a.missed && live < count ? missed_launches(tensors, count, a, st) : GS_OK;
}

extern "C" int gs_moments8_quantize(const gs_tensor* tensors, int64_t count, uint8_t* m, uint8_t* v, uint8_t* m_exp,
                                    uint8_t* v_exp, int64_t step, gs_stream_t stream) {
    int64_t live;
    GS_TRY(check_tensors("moments8_quantize", tensors, count, kNeedParam | kNeedGrad, live));
    if (live == 0) return GS_OK;
    GS_REQUIRE(m && v && m_exp && v_exp, "moments8_quantize: null pointer");
    GS_REQUIRE(aligned16(m) && aligned16(v), "moments8_quantize: codes must be 16-byte aligned");
    const uint32_t word = (uint32_t)step * kDitherStep;
    const cudaStream_t st = (cudaStream_t)stream;
    return count <= kSmallTable ? quantize_launches<kSmallTable>(tensors, count, live, m, v, m_exp, v_exp, word, st)
                                : quantize_launches<kLargeTable>(tensors, count, live, m, v, m_exp, v_exp, word, st);
}

extern "C" int gs_moments8_dequantize(const uint8_t* m, const uint8_t* v, const uint8_t* m_exp, const uint8_t* v_exp,
                                      int64_t n, int out_type, void* m_out, void* v_out, gs_stream_t stream) {
    GS_REQUIRE(n >= 0 && n % GS_MOMENT_BLOCK == 0 && n / kChunk < 0x7fffffff,
               "moments8_dequantize: the slab has whole blocks of %d elements", GS_MOMENT_BLOCK);
    GS_REQUIRE(out_type == GS_F32 || out_type == GS_BF16, "moments8_dequantize: values are float32 or bfloat16");
    if (n == 0) return GS_OK;
    GS_REQUIRE(m && v && m_exp && v_exp && m_out && v_out, "moments8_dequantize: null pointer");
    GS_REQUIRE(aligned16(m) && aligned16(v) && aligned16(m_out) && aligned16(v_out),
               "moments8_dequantize: buffers must be 16-byte aligned");
    auto k = out_type == GS_F32 ? moments8_dequantize_kernel<GS_F32> : moments8_dequantize_kernel<GS_BF16>;
    return launch_pdl("moments8_dequantize_kernel", k, dim3((unsigned)((n + kChunk - 1) / kChunk)),
                      dim3(kMultiThreads), (cudaStream_t)stream, m, v, m_exp, v_exp, n, m_out, v_out);
}
