// The global norm of many gradients and their clipping by it.
//
//   norm = |grad_scale| sqrt(sum over all tensors of g^2)
//   g'   = g * max_norm / norm   when norm > max_norm
//
// The squares are formed and summed in 64 bits: a norm over tens of millions of
// elements is then correct to float32's last bit whatever the order, and finite in
// float32 wherever it lies in float32's range.  The order is fixed too (each block
// writes one partial sum, every consumer adds them by the same tree), so a run
// repeats bit for bit.  Finding the norm has to read every gradient before the
// first may be scaled; only gradients that still lie in the 126 MB L2 are not read
// from memory twice.  59M float32: norm 36 us (of measured copy rate: 100 %), norm
// and clipping into other tensors 120 us (three passes: 90 %), in place 116 us;
// bfloat16 is held up by the conversions to 64 bits (norm 22 us, 81 %).
#include <math.h>

#include "multi_tensor.cuh"

namespace gs {

// Long groups: a block's share is mostly one piece.  With short ones all blocks move
// through the memory together, and reads and writes meet in the same DRAM banks more
// often.  Norm and clipping into other tensors at ten random places, medians: 59M
// float32 137 us, 137 with groups of 8 chunks, 145 with single ones; 118M bfloat16 142,
// 151 and 177.
constexpr int kNormBlocksPerSm = 4, kNormGroup = 64;
constexpr int kClipBlocksPerSm = 4, kClipGroup = 64;

__device__ __forceinline__ double sum_squares8(const float (&x)[8]) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fma((double)x[k], (double)x[k], s);
    return s;
}

// Whole chunks, several at a time: one chunk's 16 or 32 bytes a thread are too few
// in flight for the memory's latency.  What is read stays in L2 where it can: the
// clipping or the step reads it again.
template <bool kWide>
__device__ __forceinline__ void norm_chunks(const TensorEntry& e, int64_t& i, int& chunks, double& sum) {
    constexpr int kTogether = 4;
    for (; chunks >= kTogether && i + (kTogether - 1) * kChunk + kPerThread <= e.n; chunks -= kTogether) {
        const char* at = static_cast<const char*>(e.grad) + i * (kWide ? 4 : 2);
        Raw8 r[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) r[k] = load_raw8<kWide, false>(at + k * kChunk * (kWide ? 4 : 2));
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            float g[8];
            unpack8<kWide>(r[k], e.grad_type, g);
            sum += sum_squares8(g);
        }
        i += kTogether * kChunk;
    }
}

template <int kCap>
__global__ void __launch_bounds__(kMultiThreads) grad_norm_kernel(const __grid_constant__ TensorTable<kCap> tab,
                                                                  double* partials) {
    pdl_wait();
    double sum = 0.0;
    Segments<kCap> seg(tab);
    int chunks;
    int64_t i;
    while (seg.next(chunks, i)) {
        const TensorEntry& e = tab.e[seg.tensor];
        i += threadIdx.x * kPerThread;
        float g[8];
        if (e.grad_vec) {
            if (e.grad_type == GS_F32)
                norm_chunks<true>(e, i, chunks, sum);
            else
                norm_chunks<false>(e, i, chunks, sum);
        }
        // a warp as one: its lanes may load for one another
        for (; chunks > 0 && i - (threadIdx.x & 31) * kPerThread < e.n; --chunks, i += kChunk) {
            load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, e.grad_vec, g);
            sum += sum_squares8(g);
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// Whole chunks, 32 bytes of gradients a thread in flight: with more of them reads
// and writes disturb one another in DRAM (norm and clipping of 236M float32: 460 us,
// and 499 with twice that).
template <bool kWide>
__device__ __forceinline__ void clip_chunks(const TensorEntry& e, float f, int64_t& i, int& chunks) {
    constexpr int kTogether = kWide ? 1 : 2;
    for (; chunks >= kTogether && i + (kTogether - 1) * kChunk + kPerThread <= e.n; chunks -= kTogether) {
        const char* at = static_cast<const char*>(e.grad) + i * (kWide ? 4 : 2);
        Raw8 r[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) r[k] = load_raw8<kWide>(at + k * kChunk * (kWide ? 4 : 2));
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            float g[8];
            unpack8<kWide>(r[k], e.grad_type, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = __fmul_rn(g[j], f);
            if (e.param_type == GS_F32)
                store_vec8<true, true>(static_cast<float*>(e.param) + i + k * kChunk, GS_F32, g);
            else
                store_vec8<false, true>(static_cast<uint16_t*>(e.param) + i + k * kChunk, e.param_type, g);
        }
        i += kTogether * kChunk;
    }
}

template <int kCap>
__global__ void __launch_bounds__(kMultiThreads) grad_clip_kernel(const __grid_constant__ TensorTable<kCap> tab,
                                                                  const double* partials, int64_t num_partials,
                                                                  double max_norm, float* norm_out) {
    __shared__ float factor;
    pdl_wait();
    const double sq = sum_partials(partials, num_partials);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sq);
        // a norm that is not finite in float32 leaves the gradients as they are
        factor = norm > max_norm && isfinite((float)norm) ? (float)(max_norm / norm) : 1.0f;
        if (blockIdx.x == 0 && norm_out) *norm_out = (float)norm;
    }
    __syncthreads();
    const float f = factor;
    Segments<kCap> seg(tab);
    int chunks;
    int64_t i;
    while (seg.next(chunks, i)) {
        const TensorEntry& e = tab.e[seg.tensor];
        if (f == 1.0f && e.param == e.grad) continue;  // in place and not clipped
        i += threadIdx.x * kPerThread;
        float g[8];
        if (e.grad_vec && e.param_vec) {
            if (e.grad_type == GS_F32)
                clip_chunks<true>(e, f, i, chunks);
            else
                clip_chunks<false>(e, f, i, chunks);
        }
        // a warp as one: its lanes may load for one another
        for (; chunks > 0 && i - (threadIdx.x & 31) * kPerThread < e.n; --chunks, i += kChunk) {
            load_each8(e.grad, i, e.n, e.cols, e.grad_stride, e.grad_type, e.grad_vec, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = __fmul_rn(g[j], f);
            store_each8(e.param, i, e.n, e.cols, e.param_stride, e.param_type, e.param_vec, g);
        }
    }
}

template <int kCap>
static int norm_launches(const gs_tensor* t, int64_t count, int64_t left, double* partials, int64_t capacity,
                         int64_t* written, cudaStream_t stream) {
    TensorTable<kCap> tab;
    int64_t done = 0;
    for (int64_t at = 0; left > 0;) {
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        const int grid = table_grid(tab, kNormBlocksPerSm, kNormGroup);
        if (done + grid > capacity)
            return set_error(GS_ERR_CAPACITY, "grad_norm: %lld partial sums do not fit", (long long)capacity);
        double* out = partials + done;
        void* args[] = {&tab, &out};
        GS_TRY(launch_table("grad_norm_kernel", (const void*)grad_norm_kernel<kCap>, grid, stream, args));
        done += grid;
    }
    *written = done;
    return GS_OK;
}

template <int kCap>
static int clip_launches(const gs_tensor* t, int64_t count, int64_t left, const double* partials,
                         int64_t num_partials, double max_norm, float* norm_out, cudaStream_t stream) {
    TensorTable<kCap> tab;
    for (int64_t at = 0; left > 0;) {
        at = fill_table(tab, t, at, count);
        left -= tab.count;
        void* args[] = {&tab, &partials, &num_partials, &max_norm, &norm_out};
        GS_TRY(launch_table("grad_clip_kernel", (const void*)grad_clip_kernel<kCap>,
                            table_grid(tab, kClipBlocksPerSm, kClipGroup), stream, args));
    }
    return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" int64_t gs_grad_norm_max_partials(int64_t count) {
    // at most one wave of blocks for every table of tensors
    if (count <= 0) return 0;
    const int64_t cap = count <= kSmallTable ? kSmallTable : kLargeTable;
    return (count + cap - 1) / cap * std::min((int64_t)sm_count() * kNormBlocksPerSm, (int64_t)kMaxGrid);
}

extern "C" int gs_grad_norm_partials(const gs_tensor* tensors, int64_t count, double* partials, int64_t capacity,
                                     int64_t* num_partials, gs_stream_t stream) {
    GS_REQUIRE(num_partials, "grad_norm: null count");
    *num_partials = 0;
    int64_t live;
    GS_TRY(check_tensors("grad_norm", tensors, count, kNeedGrad | kMayMiss, live));
    if (live == 0) return GS_OK;
    GS_REQUIRE(partials && capacity > 0, "grad_norm: null partial sums");
    const cudaStream_t st = (cudaStream_t)stream;
    return count <= kSmallTable
               ? norm_launches<kSmallTable>(tensors, count, live, partials, capacity, num_partials, st)
               : norm_launches<kLargeTable>(tensors, count, live, partials, capacity, num_partials, st);
}

extern "C" int gs_clip_gradients(const gs_tensor* tensors, int64_t count, const double* partials,
                                 int64_t num_partials, double max_norm, float* norm_out, gs_stream_t stream) {
    GS_REQUIRE(max_norm > 0.0, "clip_gradients: max_norm must be positive");
    GS_REQUIRE(num_partials >= 0, "clip_gradients: bad partial count");
    int64_t live;
    GS_TRY(check_tensors("clip_gradients", tensors, count, kNeedParam | kNeedGrad, live));
    if (live == 0) return GS_OK;
    GS_REQUIRE(partials, "clip_gradients: null partial sums");
    const cudaStream_t st = (cudaStream_t)stream;
    return count <= kSmallTable
               ? clip_launches<kSmallTable>(tensors, count, live, partials, num_partials, max_norm, norm_out, st)
               : clip_launches<kLargeTable>(tensors, count, live, partials, num_partials, max_norm, norm_out, st);
}
