// One launch over many tensors: the table of tensors that a kernel takes as a
// parameter, the walk of a block over its share of their elements, and loads and
// stores of eight consecutive elements of a tensor as float32.
//
// The table travels in the kernel's parameters (at most 32,764 bytes), so a call
// needs no copy to the device, owns no memory and can be captured into a graph.
// Elements are handled in chunks of kChunk; the chunks of all tensors form one
// sequence (``first`` holds each tensor's place in it) and every block takes an
// equal, contiguous share, so one large tensor and many tiny ones balance alike.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gs {

constexpr int kMultiThreads = 256;
constexpr int kPerThread = 8;
constexpr int kChunk = kMultiThreads * kPerThread;

struct TensorEntry {
    void* param;
    void* grad;
    int64_t n, state;
    int64_t cols, param_stride, grad_stride;
    double lr_scale, decay;
    int16_t param_type, grad_type;
    int8_t param_vec, grad_vec;  // dense and aligned for 16-byte accesses
};

template <int kCap>
struct TensorTable {
    TensorEntry e[kCap];
    int32_t first[kCap + 1];
    int32_t count;
};

// Table sizes: a small one for the handful of tensors of a scene (a 2 KB
// parameter block), and the largest that fits the parameter space with room for
// a kernel's other arguments.
constexpr int kSmallTable = 24;
constexpr int kLargeTable = 368;

// ---------------------------------------------------------------- device side
struct Raw8 {
    uint4 a, b;
};

__device__ __forceinline__ Raw8 load_raw8(const void* base, int64_t i, int type) {
    Raw8 r;
    if (type == GS_F32) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
        r.a = __ldcs(p);
        r.b = __ldcs(p + 1);
    } else {
        r.a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i));
        r.b = make_uint4(0, 0, 0, 0);
    }
    return r;
}

__device__ __forceinline__ float2 unpack2(uint32_t w, int type) {
    if (type == GS_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ void unpack8(const Raw8& r, int type, float (&x)[8]) {
    if (type == GS_F32) {
        x[0] = __uint_as_float(r.a.x);
        x[1] = __uint_as_float(r.a.y);
        x[2] = __uint_as_float(r.a.z);
        x[3] = __uint_as_float(r.a.w);
        x[4] = __uint_as_float(r.b.x);
        x[5] = __uint_as_float(r.b.y);
        x[6] = __uint_as_float(r.b.z);
        x[7] = __uint_as_float(r.b.w);
    } else {
        const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2(w[k], type);
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {
    if (type == GS_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void store_vec8(void* base, int64_t i, int type, const float (&x)[8]) {
    if (type == GS_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
        __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i),
               make_uint4(pack2(x[0], x[1], type), pack2(x[2], x[3], type), pack2(x[4], x[5], type),
                          pack2(x[6], x[7], type)));
    }
}

__device__ __forceinline__ float load_one(const void* base, int64_t off, int type) {
    if (type == GS_F32) return static_cast<const float*>(base)[off];
    if (type == GS_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[off]);
    return __half2float(static_cast<const __half*>(base)[off]);
}

__device__ __forceinline__ void store_one(void* base, int64_t off, int type, float x) {
    if (type == GS_F32)
        static_cast<float*>(base)[off] = x;
    else if (type == GS_BF16)
        static_cast<__nv_bfloat16*>(base)[off] = __float2bfloat16_rn(x);
    else
        static_cast<__half*>(base)[off] = __float2half_rn(x);
}

// Walks the storage offsets of consecutive elements of a tensor whose rows of
// ``cols`` elements lie ``stride`` apart.
struct RowWalk {
    int64_t off, col, cols, skip;
    __device__ __forceinline__ RowWalk(int64_t i, int64_t cols_, int64_t stride) : cols(cols_), skip(stride - cols_) {
        const int64_t row = (i | cols_) >> 32 ? i / cols_ : (int64_t)((uint32_t)i / (uint32_t)cols_);
        col = i - row * cols_;
        off = row * stride + col;
    }
    __device__ __forceinline__ void next() {
        ++off;
        if (++col == cols) {
            col = 0;
            off += skip;
        }
    }
};

// Elements [i, i + 8) one by one: ragged ends, strided rows, odd alignment.
__device__ __forceinline__ void load_each8(const void* base, int64_t i, int64_t n, int64_t cols, int64_t stride,
                                           int type, float (&x)[8]) {
    RowWalk w(i, cols, stride);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        x[k] = i + k < n ? load_one(base, w.off, type) : 0.0f;
        w.next();
    }
}

__device__ __forceinline__ void store_each8(void* base, int64_t i, int64_t n, int64_t cols, int64_t stride, int type,
                                            const float (&x)[8]) {
    RowWalk w(i, cols, stride);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (i + k < n) store_one(base, w.off, type, x[k]);
        w.next();
    }
}

// The tensor that chunk c belongs to.
template <int kCap>
__device__ __forceinline__ int find_tensor(const TensorTable<kCap>& tab, int c) {
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// This block's chunks [begin, end).
template <int kCap>
__device__ __forceinline__ void block_share(const TensorTable<kCap>& tab, int& begin, int& end) {
    const int64_t total = tab.first[tab.count];
    begin = (int)(total * blockIdx.x / gridDim.x);
    end = (int)(total * (blockIdx.x + 1) / gridDim.x);
}

// Sum of ``n`` doubles by the whole block, the same in every thread and in every
// block that sums them (a fixed order).  Ends with the shared array free.
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[kMultiThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kMultiThreads / 32; ++k) s += part[k];
    __syncthreads();
    return s;
}

__device__ __forceinline__ double sum_partials(const double* partials, int64_t n) {
    double x = 0.0;
    for (int64_t k = threadIdx.x; k < n; k += kMultiThreads) x += partials[k];
    return block_sum(x);
}

// ---------------------------------------------------------------- host side
inline int type_bytes(int type) { return type == GS_F32 ? 4 : 2; }

// Whether elements can be moved 16 bytes at a time from a multiple of 8 on.
inline bool can_vector(const void* p, int64_t n, int64_t cols, int64_t stride) {
    return (cols >= n || stride == cols) && aligned16(p);
}

enum { kNeedParam = 1, kNeedGrad = 2 };

// Checks the caller's entries (before anything is launched).
inline int check_tensors(const char* what, const gs_tensor* t, int64_t count, int need) {
    GS_REQUIRE(count >= 0, "%s: negative tensor count", what);
    GS_REQUIRE(count == 0 || t, "%s: null tensor list", what);
    for (int64_t k = 0; k < count; ++k) {
        const gs_tensor& e = t[k];
        GS_REQUIRE(e.n >= 0 && e.n <= ((int64_t)1 << 40), "%s: tensor %lld: bad element count %lld", what, (long long)k,
                   (long long)e.n);
        if (e.n == 0) continue;
        GS_REQUIRE(e.cols > 0, "%s: tensor %lld: bad row length", what, (long long)k);
        GS_REQUIRE(e.state >= 0 && e.state % GS_MOMENT_BLOCK == 0,
                   "%s: tensor %lld: the state offset must be a multiple of %d", what, (long long)k, GS_MOMENT_BLOCK);
        for (int q = 0; q < 2; ++q) {
            if (!(need & (q ? kNeedGrad : kNeedParam))) continue;
            const void* p = q ? e.grad : e.param;
            const int type = q ? e.grad_type : e.param_type;
            const int64_t stride = q ? e.grad_stride : e.param_stride;
            const char* name = q ? "grad" : "param";
            GS_REQUIRE(p, "%s: tensor %lld: null %s", what, (long long)k, name);
            GS_REQUIRE(type == GS_F32 || type == GS_BF16 || type == GS_F16, "%s: tensor %lld: unknown %s type %d", what,
                       (long long)k, name, type);
            GS_REQUIRE(reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0, "%s: tensor %lld: misaligned %s", what,
                       (long long)k, name);
            GS_REQUIRE(stride >= e.cols, "%s: tensor %lld: %s row stride below the row length", what, (long long)k,
                       name);
        }
    }
    return GS_OK;
}

// Fills a table with up to kCap non-empty tensors from t[at]; returns the next place.
template <int kCap>
inline int64_t fill_table(TensorTable<kCap>& tab, const gs_tensor* t, int64_t at, int64_t count) {
    int k = 0;
    int64_t chunks = 0;
    for (; at < count && k < kCap; ++at) {
        const gs_tensor& s = t[at];
        if (s.n == 0) continue;
        const int64_t c = (s.n + kChunk - 1) / kChunk;
        if (chunks + c > 0x7fffffff) break;
        TensorEntry& e = tab.e[k];
        e.param = s.param;
        e.grad = const_cast<void*>(s.grad);
        e.n = s.n;
        e.state = s.state;
        e.cols = s.cols;
        e.param_stride = s.param_stride;
        e.grad_stride = s.grad_stride;
        e.lr_scale = s.lr_scale;
        e.decay = s.decay;
        e.param_type = (int16_t)s.param_type;
        e.grad_type = (int16_t)s.grad_type;
        e.param_vec = can_vector(s.param, s.n, s.cols, s.param_stride);
        e.grad_vec = can_vector(s.grad, s.n, s.cols, s.grad_stride);
        tab.first[k] = (int32_t)chunks;
        chunks += c;
        ++k;
    }
    tab.first[k] = (int32_t)chunks;
    tab.count = k;
    return at;
}

inline int64_t live_tensors(const gs_tensor* t, int64_t count) {
    int64_t k = 0;
    for (int64_t i = 0; i < count; ++i) k += t[i].n > 0;
    return k;
}

// Blocks for a table: a wave of resident blocks, or fewer when there is less work.
template <int kCap>
inline int table_grid(const TensorTable<kCap>& tab, int blocks_per_sm) {
    const int64_t most = (int64_t)sm_count() * blocks_per_sm;
    const int64_t chunks = tab.first[tab.count];
    return (int)(chunks < most ? chunks : most);
}

// Launch with programmatic stream serialisation (the kernel begins with
// pdl_wait()); arguments by address, since a table is large.
inline int launch_table(const char* what, const void* kernel, int grid, cudaStream_t stream, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kMultiThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
    note_launches(1);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(GS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    }
    return GS_OK;
}

}  // namespace gs
