// AdamW over many tensors in one launch, moments in 32 bits or in 8, and the
// conversions between the two forms.
//
// For element p of a tensor with gradient g, at step t (both counted on the
// device, so a captured step can be replayed):
//   g' = c g                       c: grad_scale, times max_norm / norm when clipped
//   m' = b1 m + (1 - b1) g'        v' = b2 v + (1 - b2) g'^2
//   p' = (1 - lr wd) p - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// The moments' operations are rounded to float32 one by one (no fused multiply-
// add), which fixes them bit for bit; all load paths give the same results.  t, the bias corrections, the norm and the factors
// made of them are formed in 64 bits and rounded once.
#include <float.h>
#include <math.h>

#include "moments8.cuh"
#include "multi_tensor.cuh"

namespace gs {

constexpr int kAdamWBlocksPerSm = 3;

struct AdamWArgs {
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    float* master;
    int64_t* ctl;           // [0] steps taken, [1] blocks that have read it
    const float* lr_dev;    // overrides lr
    const double* partials;
    float* norm_out;
    int64_t num_partials;
    double lr, log2_b1, log2_b2, grad_scale, max_norm;
    float b1, b2, omb1, omb2, eps;
    int advance;            // the step's last launch counts the step
};

struct AdamWShared {
    double lr, inv_bc1;
    float gscale, inv_sqrt_bc2;
    uint32_t step_word;
    int64_t t;
    int skip;
};

// What every element of the step shares.  Each block sums the norm's partials
// itself (a few hundred doubles in a fixed order), which needs no launch
// between the norm and the step; the bias corrections are formed by other warps
// meanwhile (beta^t = 2^(t log2 beta), in 64 bits).
__device__ __forceinline__ void adamw_prologue(const AdamWArgs& a, AdamWShared& sh) {
    double sq = 0.0;
    if (a.partials) sq = sum_partials(a.partials, a.num_partials);
    const int64_t t = *reinterpret_cast<volatile int64_t*>(a.ctl) + 1;
    if (threadIdx.x == 0) {
        double scale = a.grad_scale;
        bool skip = false;
        if (a.partials) {
            const double norm = fabs(a.grad_scale) * sqrt(sq);
            skip = !isfinite((float)norm);
            if (norm > a.max_norm) scale *= a.max_norm / norm;
            if (blockIdx.x == 0 && a.norm_out) *a.norm_out = (float)norm;
        }
        sh.skip = skip;
        sh.gscale = (float)scale;
        sh.lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
        sh.step_word = (uint32_t)t * kDitherStep;
    } else if (threadIdx.x == 32) {
        sh.inv_bc1 = 1.0 / (1.0 - exp2((double)t * a.log2_b1));
    } else if (threadIdx.x == 64) {
        sh.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - exp2((double)t * a.log2_b2)));
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

// The moments, every operation rounded by itself.
__device__ __forceinline__ void moments_update(float g, float& m, float& v, const AdamWArgs& a) {
    m = __fadd_rn(__fmul_rn(a.b1, m), __fmul_rn(a.omb1, g));
    v = __fadd_rn(__fmul_rn(a.b2, v), __fmul_rn(a.omb2, __fmul_rn(g, g)));
}

// The parameter, with the hardware's approximate square root and reciprocal: 2
// ulp each on the step, far below the rounding of the parameter it moves.  The
// rounded forms take a slow path where m or v is a denormal, which is where the
// moments of long unseen Gaussians end (0.9^800 of a gradient): a step over a
// scene half of which is unseen took 561 us with them and 269 us without.
__device__ __forceinline__ float param_update(float p, float m, float v, float inv_sqrt_bc2, float step, float keep,
                                              float eps) {
    float root, inv;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
    const float denom = fmaf(root, inv_sqrt_bc2, eps);  // eps is a normal number, so denom is
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(denom));
    return fmaf(-step, m * inv, p * keep);
}

template <int kBits, int kCap>
__global__ void __launch_bounds__(kMultiThreads, kAdamWBlocksPerSm) adamw_kernel(
    const __grid_constant__ TensorTable<kCap> tab, const __grid_constant__ AdamWArgs a) {
    __shared__ AdamWShared sh;
    pdl_wait();
    int c, end;
    block_share(tab, c, end);
    int ti = find_tensor(tab, c);
    float step = 0.0f, keep = 0.0f;
    // the grid has at most one block per chunk, so every block has a first chunk
    for (int seen = -1; c < end; ++c) {
        while (c >= tab.first[ti + 1]) ++ti;
        const TensorEntry& e = tab.e[ti];
        const int64_t i = (int64_t)(c - tab.first[ti]) * kChunk + threadIdx.x * kPerThread;
        const int64_t s = e.state + i;
        // the state has whole blocks of 256, so a warp is inside or outside as one
        const bool inside = i - (threadIdx.x & 31) * kPerThread < e.n;
        const bool whole = i + kPerThread <= e.n;
        const bool masters = a.master != nullptr && e.param_type != GS_F32;
        const bool vg = whole && e.grad_vec, vp = whole && e.param_vec;
        Raw8 rp, rg, rm, rv;
        uint2 cm, cv;
        uint32_t em = 0, ev = 0;
        if (inside) {
            if (kBits == 32) {
                rm = load_raw8(a.m, s, GS_F32);
                rv = load_raw8(a.v, s, GS_F32);
            } else {
                cm = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + s));
                cv = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + s));
                em = a.m_exp[s / GS_MOMENT_BLOCK];
                ev = a.v_exp[s / GS_MOMENT_BLOCK];
            }
            if (vg) rg = load_raw8(e.grad, i, e.grad_type);
            if (masters)
                rp = load_raw8(a.master, s, GS_F32);
            else if (vp)
                rp = load_raw8(e.param, i, e.param_type);
        }
        if (ti != seen) {
            // the first chunk's loads are on their way while the block forms what the step shares
            if (seen < 0) {
                adamw_prologue(a, sh);
                if (sh.skip) return;
            }
            const double lr = sh.lr * e.lr_scale;
            step = (float)(lr * sh.inv_bc1);
            keep = (float)(1.0 - lr * e.decay);
            seen = ti;
        }
        if (!inside) continue;
        float p[8], g[8], m[8], v[8];
        if (vg)
            unpack8(rg, e.grad_type, g);
        else
            load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, g);
        if (kBits == 32) {
            unpack8(rm, GS_F32, m);
            unpack8(rv, GS_F32, v);
        } else {
            decode_m8(cm, em, m);
            decode_v8(cv, ev, v);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) moments_update(__fmul_rn(g[k], sh.gscale), m[k], v[k], a);
        if (masters)
            unpack8(rp, GS_F32, p);
        else if (vp)
            unpack8(rp, e.param_type, p);
        else
            load_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, p);
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = param_update(p[k], m[k], v[k], sh.inv_sqrt_bc2, step, keep, a.eps);
        if (masters) store_vec8(a.master, s, GS_F32, p);
        if (vp)
            store_vec8(e.param, i, e.param_type, p);
        else
            store_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, p);
        if (kBits == 32) {
            store_vec8(a.m, s, GS_F32, m);
            store_vec8(a.v, s, GS_F32, v);
        } else {
            store_moments8<false>(m, v, (uint32_t)i, sh.step_word, static_cast<uint8_t*>(a.m) + s,
                                  static_cast<uint8_t*>(a.v) + s, a.m_exp + s / GS_MOMENT_BLOCK,
                                  a.v_exp + s / GS_MOMENT_BLOCK);
        }
    }
}

// m (the entries' param) and v (their grad) of any type -> the 8-bit form, with
// step t's offsets.
template <int kCap>
__global__ void __launch_bounds__(kMultiThreads) moments8_quantize_kernel(const __grid_constant__ TensorTable<kCap> tab,
                                                                          uint8_t* mc, uint8_t* vc, uint8_t* me,
                                                                          uint8_t* ve, uint32_t step_word) {
    pdl_wait();
    int c, end;
    block_share(tab, c, end);
    if (c >= end) return;
    int ti = find_tensor(tab, c);
    for (; c < end; ++c) {
        while (c >= tab.first[ti + 1]) ++ti;
        const TensorEntry& e = tab.e[ti];
        const int64_t i = (int64_t)(c - tab.first[ti]) * kChunk + threadIdx.x * kPerThread;
        const int64_t s = e.state + i;
        if (i - (threadIdx.x & 31) * kPerThread >= e.n) continue;
        const bool whole = i + kPerThread <= e.n;
        float m[8], v[8];
        Raw8 rm, rv;
        const bool vm = whole && e.param_vec, vv = whole && e.grad_vec;
        if (vm) rm = load_raw8(e.param, i, e.param_type);
        if (vv) rv = load_raw8(e.grad, i, e.grad_type);
        if (vm)
            unpack8(rm, e.param_type, m);
        else
            load_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, m);
        if (vv)
            unpack8(rv, e.grad_type, v);
        else
            load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, v);
        store_moments8<true>(m, v, (uint32_t)i, step_word, mc + s, vc + s, me + s / GS_MOMENT_BLOCK,
                       ve + s / GS_MOMENT_BLOCK);
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

template <int kCap>
static int adamw_launches(const gs_tensor* t, int64_t count, int bits, AdamWArgs a, cudaStream_t stream) {
    TensorTable<kCap> tab;
    int64_t left = live_tensors(t, count);
    for (int64_t at = 0; left > 0;) {
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        a.advance = left == 0;
        void* args[] = {&tab, &a};
        const void* k = bits == 32 ? (const void*)adamw_kernel<32, kCap> : (const void*)adamw_kernel<8, kCap>;
        GS_TRY(launch_table("adamw_kernel", k, table_grid(tab, kAdamWBlocksPerSm), stream, args));
    }
    return GS_OK;
}

template <int kCap>
static int quantize_launches(const gs_tensor* t, int64_t count, uint8_t* m, uint8_t* v, uint8_t* me, uint8_t* ve,
                             uint32_t step_word, cudaStream_t stream) {
    TensorTable<kCap> tab;
    int64_t left = live_tensors(t, count);
    for (int64_t at = 0; left > 0;) {
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        void* args[] = {&tab, &m, &v, &me, &ve, &step_word};
        GS_TRY(launch_table("moments8_quantize_kernel", (const void*)moments8_quantize_kernel<kCap>,
                            table_grid(tab, 4), stream, args));
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
    GS_REQUIRE(isfinite(set->grad_scale), "adamw: grad_scale must be finite");
    GS_REQUIRE(set->lr_device || isfinite(set->lr), "adamw: lr must be finite");
    GS_REQUIRE(!set->norm_partials || (set->num_partials >= 0 && set->max_norm > 0.0),
               "adamw: clipping needs a partial count and a positive max_norm");
    GS_TRY(check_tensors("adamw", tensors, count, kNeedParam | kNeedGrad));
    if (live_tensors(tensors, count) == 0) return GS_OK;
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
    return count <= kSmallTable ? adamw_launches<kSmallTable>(tensors, count, state->bits, a, st)
                                : adamw_launches<kLargeTable>(tensors, count, state->bits, a, st);
}

extern "C" int gs_moments8_quantize(const gs_tensor* tensors, int64_t count, uint8_t* m, uint8_t* v, uint8_t* m_exp,
                                    uint8_t* v_exp, int64_t step, gs_stream_t stream) {
    GS_TRY(check_tensors("moments8_quantize", tensors, count, kNeedParam | kNeedGrad));
    if (live_tensors(tensors, count) == 0) return GS_OK;
    GS_REQUIRE(m && v && m_exp && v_exp, "moments8_quantize: null pointer");
    GS_REQUIRE(aligned16(m) && aligned16(v), "moments8_quantize: codes must be 16-byte aligned");
    const uint32_t word = (uint32_t)step * kDitherStep;
    const cudaStream_t st = (cudaStream_t)stream;
    return count <= kSmallTable ? quantize_launches<kSmallTable>(tensors, count, m, v, m_exp, v_exp, word, st)
                                : quantize_launches<kLargeTable>(tensors, count, m, v, m_exp, v_exp, word, st);
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
