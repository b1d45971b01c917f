// One launch over many tensors: the table of tensors that a kernel takes as a
// parameter, the walk of a block over its share of their elements, and loads and
// stores of eight consecutive elements of a tensor as float32.
//
// The table travels in the kernel's parameters (at most 32,764 bytes), so a call
// needs no copy to the device, owns no memory and can be captured into a graph.
// Elements are handled in chunks of kChunk; the chunks of all tensors form one
// sequence (``first`` holds each tensor's place in it) of which every block takes
// equal shares, so one large tensor and many tiny ones balance alike.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

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
    int8_t param_vec, grad_vec;  // dense and aligned for accesses to eight elements
    uint16_t place;              // in the caller's list, counted from the table's first tensor
};

// Table sizes: a small one for the handful of tensors of a scene (a 2 KB
// parameter block), and the largest that fits the parameter space with room for
// a kernel's other arguments.
constexpr int kSmallTable = 24;
constexpr int kLargeTable = 360;
constexpr int kMaxGrid = 640;  // four blocks on each of 160 SMs

template <int kCap>
struct TensorTable {
    TensorEntry e[kCap];
    int32_t first[kCap + 1];
    int32_t count;
    int32_t group, groups;  // chunks that a block takes at a time, and how many such groups there are
    int32_t all_vec;        // every tensor of the call is dense and aligned
    // The tensor that each block begins in: a search through a large table costs a block several dependent reads of
    // parameters that no one has read yet.  (A small table is searched.)
    uint16_t begin[kCap > kSmallTable ? kMaxGrid : 1];
};

// ---------------------------------------------------------------- device side
// Eight consecutive elements as they lie in memory: 32 bytes of float32 or 16.
// (One 256-bit access for float32 instead of two of 128 measured the same in the
// steps and slower in the moments' quantization, 120 us against 104 for 59M.)
struct Raw8 {
    uint4 a, b;
};

// kStream: not expected to be read again soon (evicted first from L2).
template <bool kStream>
__device__ __forceinline__ uint4 load16(const uint4* p) {
    return kStream ? __ldcs(p) : *p;
}

// kWide: float32; else the two 16-bit types.
template <bool kWide, bool kStream = true>
__device__ __forceinline__ Raw8 load_raw8(const void* p) {
    Raw8 r;
    r.a = load16<kStream>(static_cast<const uint4*>(p));
    r.b = kWide ? load16<kStream>(static_cast<const uint4*>(p) + 1) : make_uint4(0, 0, 0, 0);
    return r;
}

__device__ __forceinline__ Raw8 load_raw8(const void* base, int64_t i, int type) {
    return type == GS_F32 ? load_raw8<true>(static_cast<const float*>(base) + i)
                          : load_raw8<false>(static_cast<const uint16_t*>(base) + i);
}

template <bool kWide>
__device__ __forceinline__ void unpack8(const Raw8& r, int type, float (&x)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (kWide) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(w[k]);
    } else if (type == GS_BF16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}

__device__ __forceinline__ void unpack8(const Raw8& r, int type, float (&x)[8]) {
    if (type == GS_F32)
        unpack8<true>(r, type, x);
    else
        unpack8<false>(r, type, x);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {
    if (type == GS_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool kStream>
__device__ __forceinline__ void store16(void* p, uint4 x) {
    if (kStream)
        __stcs(static_cast<uint4*>(p), x);
    else
        *static_cast<uint4*>(p) = x;
}

template <bool kWide, bool kStream = false>
__device__ __forceinline__ void store_vec8(void* p, int type, const float (&x)[8]) {
    if (kWide) {
#pragma unroll
        for (int k = 0; k < 8; k += 4)
            store16<kStream>(static_cast<float*>(p) + k,
                             make_uint4(__float_as_uint(x[k]), __float_as_uint(x[k + 1]), __float_as_uint(x[k + 2]),
                                        __float_as_uint(x[k + 3])));
    } else if (type == GS_BF16) {
        store16<kStream>(p, make_uint4(pack2(x[0], x[1], GS_BF16), pack2(x[2], x[3], GS_BF16),
                                       pack2(x[4], x[5], GS_BF16), pack2(x[6], x[7], GS_BF16)));
    } else {
        store16<kStream>(p, make_uint4(pack2(x[0], x[1], GS_F16), pack2(x[2], x[3], GS_F16),
                                       pack2(x[4], x[5], GS_F16), pack2(x[6], x[7], GS_F16)));
    }
}

__device__ __forceinline__ void store_vec8(void* base, int64_t i, int type, const float (&x)[8]) {
    if (type == GS_F32)
        store_vec8<true>(static_cast<float*>(base) + i, type, x);
    else
        store_vec8<false>(static_cast<uint16_t*>(base) + i, type, x);
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

// Storage offsets of every 32nd element of a tensor whose rows of ``cols`` elements
// lie ``stride`` apart.
struct RowWalk {
    int64_t off, col, cols, step, col_step, skip;
    __device__ __forceinline__ RowWalk(int64_t i, int64_t cols_, int64_t stride) : cols(cols_), skip(stride - cols_) {
        const int64_t row = (i | cols_) >> 32 ? i / cols_ : (int64_t)((uint32_t)i / (uint32_t)cols_);
        col = i - row * cols_;
        off = row * stride + col;
        const int rows = cols_ < 32 ? 32 / (int)cols_ : 0;
        col_step = 32 - rows * cols_;
        step = rows * stride + col_step;
    }
    __device__ __forceinline__ void next() {
        off += step;
        col += col_step;
        if (col >= cols) {
            col -= cols;
            off += skip;
        }
    }
};

// Eight consecutive elements a lane of a warp's 256, where rows or alignment rule
// wide accesses out: the warp loads and stores 32 neighbours at a time and turns
// them round in shared memory.  Every lane takes part; ``i`` is the lane's first
// element.  Loads begin in start_rows8 and are waited for in finish_rows8, so that
// two tensors' can be under way together.  (Each lane by itself, eight accesses 32
// bytes apart: a step over the columns of a pool of 1M Gaussians with dense gradients
// took 628 us, where it now takes 489.)
__device__ __forceinline__ float* warp_stage() {
    __shared__ __align__(16) float stage[kMultiThreads / 32][32 * kPerThread];
    return stage[threadIdx.x >> 5];
}

template <int kType>
__device__ __forceinline__ void gather8(const void* base, RowWalk w, int64_t left, float (&y)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        y[k] = 32 * k < left ? load_one(base, w.off, kType) : 0.0f;
        w.next();
    }
}

__device__ __forceinline__ void start_rows8(const void* base, int64_t i, int64_t n, int64_t cols, int64_t stride,
                                            int type, float (&y)[8]) {
    const int64_t first = i - (threadIdx.x & 31) * (kPerThread - 1);
    const RowWalk w(first, cols, stride);
    if (type == GS_F32)
        gather8<GS_F32>(base, w, n - first, y);
    else if (type == GS_BF16)
        gather8<GS_BF16>(base, w, n - first, y);
    else
        gather8<GS_F16>(base, w, n - first, y);
}

__device__ __forceinline__ void finish_rows8(const float (&y)[8], float (&x)[8]) {
    const int lane = threadIdx.x & 31;
    float* s = warp_stage();
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) s[32 * k + lane] = y[k];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        const float4 q = *reinterpret_cast<const float4*>(s + kPerThread * lane + k);
        x[k] = q.x;
        x[k + 1] = q.y;
        x[k + 2] = q.z;
        x[k + 3] = q.w;
    }
}

__device__ __forceinline__ void store_rows8(void* base, int64_t i, int64_t n, int64_t cols, int64_t stride, int type,
                                            const float (&x)[8]) {
    const int lane = threadIdx.x & 31;
    float* s = warp_stage();
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; k += 4)
        *reinterpret_cast<float4*>(s + kPerThread * lane + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
    __syncwarp();
    const int64_t first = i - lane * (kPerThread - 1);
    RowWalk w(first, cols, stride);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (32 * k < n - first) store_one(base, w.off, type, s[32 * k + lane]);
        w.next();
    }
}

// Dense, aligned tensors: wide accesses, and single ones at the end.
__device__ __forceinline__ void load_tail8(const void* base, int64_t i, int64_t n, int type, float (&x)[8]) {
    if (i + kPerThread <= n) {
        unpack8(load_raw8(base, i, type), type, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = i + k < n ? load_one(base, i + k, type) : 0.0f;
    }
}

__device__ __forceinline__ void store_tail8(void* base, int64_t i, int64_t n, int type, const float (&x)[8]) {
    if (i + kPerThread <= n) {
        store_vec8(base, i, type, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (i + k < n) store_one(base, i + k, type, x[k]);
        }
    }
}

// Any tensor.
__device__ __forceinline__ void load_each8(const void* base, int64_t i, int64_t n, int64_t cols, int64_t stride,
                                           int type, bool vec, float (&x)[8]) {
    if (vec) {
        load_tail8(base, i, n, type, x);
    } else {
        float y[8];
        start_rows8(base, i, n, cols, stride, type, y);
        finish_rows8(y, x);
    }
}

__device__ __forceinline__ void store_each8(void* base, int64_t i, int64_t n, int64_t cols, int64_t stride, int type,
                                            bool vec, const float (&x)[8]) {
    if (vec)
        store_tail8(base, i, n, type, x);
    else
        store_rows8(base, i, n, cols, stride, type, x);
}

// A block's way through the chunks: it takes every gridDim-th group of successive
// ones, in segments that lie in one tensor.  Neighbouring blocks work on
// neighbouring memory, which DRAM prefers to as many distant streams as there are
// blocks.
template <int kCap>
struct Segments {
    const TensorTable<kCap>& tab;
    int group, c, group_end, tensor;

    __device__ __forceinline__ explicit Segments(const TensorTable<kCap>& t) : tab(t) {
        group = blockIdx.x;  // the grid has at most one block per group
        enter();
        if (kCap > kSmallTable) {
            tensor = tab.begin[blockIdx.x];
            return;
        }
        int lo = 0, hi = tab.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (tab.first[mid] <= c)
                lo = mid;
            else
                hi = mid - 1;
        }
        tensor = lo;
    }
    __device__ __forceinline__ void enter() {
        c = group * tab.group;
        group_end = min(c + tab.group, tab.first[tab.count]);
    }
    // Moves to the next segment: ``chunks`` of tensor ``tensor`` from its element ``from`` on.
    __device__ __forceinline__ bool next(int& chunks, int64_t& from) {
        if (c == group_end) {
            group += gridDim.x;
            if (group >= tab.groups) return false;
            enter();
        }
        while (c >= tab.first[tensor + 1]) ++tensor;
        chunks = min(group_end, tab.first[tensor + 1]) - c;
        from = (int64_t)(c - tab.first[tensor]) * kChunk;
        c += chunks;
        return true;
    }
};

// Of a segment's chunks, those in which this warp's 256 elements begin inside the
// tensor (``mine``) and those in which they end inside it too (``whole``); i: the
// thread's first element.
__device__ __forceinline__ void warp_chunks(int64_t n, int64_t i, int chunks, int& mine, int& whole) {
    constexpr int kWarp = 32 * kPerThread;
    const int64_t left = n - (i - (threadIdx.x & 31) * kPerThread);
    mine = left > 0 ? (int)min((int64_t)chunks, (left - 1) / kChunk + 1) : 0;
    whole = left >= kWarp ? (int)min((int64_t)chunks, (left - kWarp) / kChunk + 1) : 0;
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

// Whether eight elements can be moved at a time from a multiple of 8 on.
inline bool can_vector(const void* p, int64_t n, int64_t cols, int64_t stride) {
    return (cols >= n || stride == cols) && aligned16(p);
}

// What a call needs of its tensors; kMayMiss: those with a null grad are passed over.
enum { kNeedParam = 1, kNeedGrad = 2, kMayMiss = 4 };

inline bool passed_over(const gs_tensor& t) { return t.n == 0 || !t.grad; }

inline bool sound_side(const void* p, int type, int64_t stride, int64_t cols) {
    return (p != nullptr) & ((unsigned)type <= GS_F16) &
           ((reinterpret_cast<uintptr_t>(p) & (type == GS_F32 ? 3u : 1u)) == 0) & (stride >= cols);
}

// Whether an entry takes part and is without a fault (one expression: a call over a few
// hundred short tensors spends more here than the device does).
inline bool sound_entry(const gs_tensor& e, int need) {
    return ((uint64_t)e.n - 1 < (uint64_t)1 << 40) & (e.cols > 0) & (e.state >= 0) & (e.state % GS_MOMENT_BLOCK == 0) &
           (!(need & kNeedParam) || sound_side(e.param, e.param_type, e.param_stride, e.cols)) &
           sound_side(e.grad, e.grad_type, e.grad_stride, e.cols);
}

// Checks the caller's entries (before anything is launched) and counts those that take part.
inline int check_tensors(const char* what, const gs_tensor* t, int64_t count, int need, int64_t& live) {
    live = 0;
    GS_REQUIRE(count >= 0, "%s: negative tensor count", what);
    GS_REQUIRE(count == 0 || t, "%s: null tensor list", what);
    for (int64_t k = 0; k < count; ++k) {
        const gs_tensor& e = t[k];
        if (sound_entry(e, need)) {
            ++live;
            continue;
        }
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
            if (q && !p && (need & kMayMiss)) continue;
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

// Fills a table with up to kCap tensors that have elements and a grad from t[at]; returns
// the next place.
template <int kCap>
inline int64_t fill_table(TensorTable<kCap>& tab, const gs_tensor* t, int64_t at, int64_t count) {
    int k = 0;
    int64_t chunks = 0;
    int64_t from = at;
    tab.all_vec = 1;
    for (; at < count && k < kCap; ++at) {
        const gs_tensor& s = t[at];
        if (passed_over(s)) continue;
        if (k == 0) from = at;
        if (at - from > 0xffff) break;
        const int64_t c = (s.n + kChunk - 1) / kChunk;
        if (chunks + c > 0x7f000000) break;
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
        e.place = (uint16_t)(at - from);
        e.param_type = (int16_t)s.param_type;
        e.grad_type = (int16_t)s.grad_type;
        e.param_vec = can_vector(s.param, s.n, s.cols, s.param_stride);
        e.grad_vec = can_vector(s.grad, s.n, s.cols, s.grad_stride);
        tab.all_vec &= e.param_vec & e.grad_vec;
        tab.first[k] = (int32_t)chunks;
        chunks += c;
        ++k;
    }
    tab.first[k] = (int32_t)chunks;
    tab.count = k;
    return at;
}

// Blocks for a table and the size of their groups: at most one wave of resident
// blocks, and groups of at most ``most_group`` chunks, of the size that lets every
// block take the same number of them.
template <int kCap>
inline int table_grid(TensorTable<kCap>& tab, int blocks_per_sm, int most_group) {
    const int64_t chunks = tab.first[tab.count];
    const int64_t wave = std::min((int64_t)sm_count() * blocks_per_sm, (int64_t)kMaxGrid);
    const int64_t rounds = (chunks + wave * most_group - 1) / (wave * most_group);
    tab.group = (int32_t)((chunks + wave * rounds - 1) / (wave * rounds));
    tab.groups = (int32_t)((chunks + tab.group - 1) / tab.group);
    const int grid = (int)(tab.groups < wave ? tab.groups : wave);
    if (kCap > kSmallTable) {
        int t = 0;
        for (int b = 0; b < grid; ++b) {
            while (tab.first[t + 1] <= b * tab.group) ++t;
            tab.begin[b] = (uint16_t)t;
        }
    }
    return grid;
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
