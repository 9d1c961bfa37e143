// clip.cu -- the 2-norm over many tensors together, and scaling them to a largest norm.
//
//   norm = sqrt(sum_t sum_e g_te^2)        out = g min(1, max_norm / norm)
//
// Bound by memory: one read for the norm, one read and one write for the scaling (the second
// read comes from L2 where the tensors fit).  The tensors' addresses travel as kernel
// parameters, so that no table is copied to the device and a graph holds the whole call.
// Measured on a B200 (copy rate 6,551 GB/s): the norm of 2 GB of fp32 0.29 ms (6,900 GB/s); 401
// tensors, 534 MB in 16 and 32 bits: norm 0.09 to 0.11 ms, scaling 0.19 ms (5,600 GB/s read and
// written), with the host's lists of pointers 0.34 ms a call.
// Squares are summed in fp64 (a square of an fp32 or bf16 value can leave fp32's range): each
// CTA writes one partial sum, and whoever needs the norm adds the partials in the same order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "engine.h"
#include "xent.h"

namespace gafime {

namespace {

constexpr int kThreads = 256;
constexpr int kGridPerSm = 8;
constexpr int kMaxGrid = 2048;
constexpr int kChunk = 16384;      // elements a CTA takes at a time
constexpr int kFewTensors = 32, kManyTensors = 1024;   // of one launch

template <int K>
struct Table {
    const void* in[K];
    void* out[K];
    int64_t size[K];
    uint32_t chunk0[K + 1];        // chunks before tensor i
    uint8_t type[K];
    int count;
};

__device__ __forceinline__ void unpack(float (&v)[4], const uint4& q, float) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(float (&v)[8], const uint4& q, __half) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(float (&v)[8], const uint4& q, __nv_bfloat16) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint4 repack(const float (&v)[4], float) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 repack(const float (&v)[8], __half) {
    uint32_t u[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 repack(const float (&v)[8], __nv_bfloat16) {
    uint32_t u[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// elements of [0, len) before the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int len) {
    return min(len, (int)((16 - (uintptr_t)p % 16) % 16 / sizeof(T)));
}

template <typename T>
__device__ double chunk_squares(const T* p, int len) {
    constexpr int V = 16 / sizeof(T);
    const int head = head_of(p, len), vecs = (len - head) / V;
    double s = 0.0;
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    #pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += kThreads) {
        float v[V];
        unpack(v, q[i], T{});
        #pragma unroll
        for (int j = 0; j < V; ++j) s = fma((double)v[j], (double)v[j], s);
    }
    const int rest = len - head - vecs * V;
    if ((int)threadIdx.x < head + rest) {
        const int e = (int)threadIdx.x < head ? threadIdx.x : head + vecs * V + threadIdx.x - head;
        const double v = (double)to_float(p[e]);
        s = fma(v, v, s);
    }
    return s;
}

template <typename T>
__device__ void chunk_scale(const T* p, T* o, int len, float f, float f2) {
    constexpr int V = 16 / sizeof(T);
    if ((uintptr_t)p % 16 != (uintptr_t)o % 16) {
        for (int e = threadIdx.x; e < len; e += kThreads) o[e] = from_float<T>(to_float(p[e]) * f2 * f);
        return;
    }
    const int head = head_of(p, len), vecs = (len - head) / V;
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
    uint4* w = reinterpret_cast<uint4*>(o + head);
    #pragma unroll 4
    for (int i = threadIdx.x; i < vecs; i += kThreads) {
        float v[V];
        unpack(v, q[i], T{});
        #pragma unroll
        for (int j = 0; j < V; ++j) v[j] = v[j] * f2 * f;
        __stcs(w + i, repack(v, T{}));
    }
    const int rest = len - head - vecs * V;
    if ((int)threadIdx.x < head + rest) {
        const int e = (int)threadIdx.x < head ? threadIdx.x : head + vecs * V + threadIdx.x - head;
        o[e] = from_float<T>(to_float(p[e]) * f2 * f);
    }
}

__device__ double block_sum(double v) {
    __shared__ double s[kThreads / 32];
    #pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    #pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) t += s[i];
    return t;   // the same in every thread
}

// the tensor of chunk c
template <int K>
__device__ __forceinline__ int tensor_of(const Table<K>& t, uint32_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.chunk0[mid] <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <int K>
__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ Table<K> t, double* part) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < t.chunk0[t.count]; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const int64_t at = (int64_t)(c - t.chunk0[i]) * kChunk;
        const int len = (int)min((int64_t)kChunk, t.size[i] - at);
        if (t.type[i] == GAFIME_TYPE_FP32)
            s += chunk_squares((const float*)t.in[i] + at, len);
        else if (t.type[i] == GAFIME_TYPE_FP16)
            s += chunk_squares((const __half*)t.in[i] + at, len);
        else
            s += chunk_squares((const __nv_bfloat16*)t.in[i] + at, len);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ double norm_of(const double* part, int parts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const double* part, int parts, float* norm) {
    const double v = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <int K>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ Table<K> t, const double* part,
                                                              int parts, float max_norm, float* norm) {
    const double v = norm_of(part, parts);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    // A norm that is not finite has no scale that would mend its tensors; nor is one past fp32, which
    // the caller sees as infinity.  A factor below fp32's normal numbers comes as two.
    const double q = isfinite((float)v) && v > (double)max_norm ? (double)max_norm / v : 1.0;
    const float f2 = q < 0x1p-126 ? 0x1p-126f : 1.f, f = (float)(q / (double)f2);
    for (uint32_t c = blockIdx.x; c < t.chunk0[t.count]; c += gridDim.x) {
        const int i = tensor_of(t, c);
        if (q == 1.0 && t.in[i] == t.out[i]) continue;
        const int64_t at = (int64_t)(c - t.chunk0[i]) * kChunk;
        const int len = (int)min((int64_t)kChunk, t.size[i] - at);
        if (t.type[i] == GAFIME_TYPE_FP32)
            chunk_scale((const float*)t.in[i] + at, (float*)t.out[i] + at, len, f, f2);
        else if (t.type[i] == GAFIME_TYPE_FP16)
            chunk_scale((const __half*)t.in[i] + at, (__half*)t.out[i] + at, len, f, f2);
        else
            chunk_scale((const __nv_bfloat16*)t.in[i] + at, (__nv_bfloat16*)t.out[i] + at, len, f, f2);
    }
}

template <int K>
void fill(Table<K>& t, const void* const* in, const int64_t* sizes, const int* types, void* const* out, int64_t i0,
          int64_t count) {
    t.count = (int)count;
    uint32_t c = 0;
    for (int64_t i = 0; i < count; ++i) {
        t.in[i] = in[i0 + i];
        t.out[i] = out ? out[i0 + i] : nullptr;
        t.size[i] = sizes[i0 + i];
        t.type[i] = (uint8_t)types[i0 + i];
        t.chunk0[i] = c;
        c += (uint32_t)((sizes[i0 + i] + kChunk - 1) / kChunk);
    }
    t.chunk0[count] = c;
}

template <int K>
cudaError_t run_clip(const void* const* in, const int64_t* sizes, const int* types, int64_t n, void* const* out,
                     float max_norm, float* norm, double* part, cudaStream_t st) {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int most = std::min(kMaxGrid, kGridPerSm * sms);
    Table<K> t;
    int parts = 0;
    for (int pass = 0; pass < (out ? 2 : 1); ++pass) {
        for (int64_t i = 0; i < n; i += K) {
            fill(t, in, sizes, types, out, i, std::min<int64_t>(K, n - i));
            const int grid = (int)std::max<uint32_t>(1, std::min<uint32_t>(t.chunk0[t.count], (uint32_t)most));
            KernelTimer kt(st, GAFIME_KERNEL_GRAD_NORM);
            if (pass == 0) {
                grad_squares_kernel<K><<<grid, kThreads, 0, st>>>(t, part + parts);
                parts += grid;
            } else {
                grad_scale_kernel<K><<<grid, kThreads, 0, st>>>(t, part, parts, max_norm, i == 0 ? norm : nullptr);
            }
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    }
    if (!out || n == 0) {
        KernelTimer kt(st, GAFIME_KERNEL_GRAD_NORM);
        grad_norm_kernel<<<1, kThreads, 0, st>>>(part, parts, norm);
        return cudaGetLastError();
    }
    return cudaSuccess;
}

// true when no written range meets another tensor's range
bool ranges_apart(const void* const* in, const int64_t* sizes, const int* types, int64_t n, void* const* out) {
    struct Range {
        uintptr_t lo, hi;
        bool written;
    };
    std::vector<Range> r;
    r.reserve(2 * n);
    for (int64_t i = 0; i < n; ++i) {
        if (sizes[i] == 0) continue;
        const size_t bytes = (size_t)sizes[i] * xent_type_size(types[i]);
        r.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + bytes, true});
        if (in[i] != out[i]) r.push_back({(uintptr_t)in[i], (uintptr_t)in[i] + bytes, false});
    }
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t end = 0, written_end = 0;   // furthest end of what came before, and of what is written of it
    for (const Range& v : r) {
        if (v.lo < written_end || (v.written && v.lo < end)) return false;
        end = std::max(end, v.hi);
        if (v.written) written_end = std::max(written_end, v.hi);
    }
    return true;
}

size_t norm_workspace(int64_t n) {
    return (size_t)std::max<int64_t>(1, (n + kManyTensors - 1) / kManyTensors) * kMaxGrid * sizeof(double);
}

}  // namespace

}  // namespace gafime

using namespace gafime;

extern "C" int gafime_grad_norm_workspace(int64_t n_tensors, size_t* bytes_out) {
    if (n_tensors < 0 || n_tensors > (1 << 24) || !bytes_out) return GAFIME_ERROR_INVALID_ARGS;
    *bytes_out = norm_workspace(n_tensors);
    return GAFIME_SUCCESS;
}

extern "C" int gafime_grad_norm(const void* const* d_tensors, const int64_t* sizes, const int* types, int64_t n_tensors,
                                void* const* d_outs, float max_norm, float* d_norm, void* d_workspace,
                                size_t workspace_bytes, void* stream) {
    if (n_tensors < 0 || n_tensors > (1 << 24) || !d_norm || (uintptr_t)d_norm % 4 || !d_workspace || (uintptr_t)d_workspace % 256 ||
        workspace_bytes < norm_workspace(n_tensors))
        return GAFIME_ERROR_INVALID_ARGS;
    if (n_tensors > 0 && (!d_tensors || !sizes || !types)) return GAFIME_ERROR_INVALID_ARGS;
    if (d_outs && !(max_norm >= 0.f && max_norm <= 3.402823466e38f)) return GAFIME_ERROR_INVALID_ARGS;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (types[i] < GAFIME_TYPE_FP32 || types[i] > GAFIME_TYPE_BF16 || sizes[i] < 0 || sizes[i] > ((int64_t)1 << 36))
            return GAFIME_ERROR_INVALID_ARGS;
        const size_t es = xent_type_size(types[i]);
        if (sizes[i] > 0 && (!d_tensors[i] || (uintptr_t)d_tensors[i] % es ||
                             (d_outs && (!d_outs[i] || (uintptr_t)d_outs[i] % es))))
            return GAFIME_ERROR_INVALID_ARGS;
    }
    int64_t chunks = 0;
    for (int64_t i = 0; i < n_tensors; ++i) chunks += (sizes[i] + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffffll) return GAFIME_ERROR_INVALID_ARGS;
    try {
        if (d_outs && !ranges_apart(d_tensors, sizes, types, n_tensors, d_outs)) return GAFIME_ERROR_INVALID_ARGS;
    } catch (...) {
        return GAFIME_ERROR_OUT_OF_MEMORY;
    }
    if (gafime_cuda_available() != 1) return GAFIME_ERROR_CUDA_NOT_AVAILABLE;
    auto run = n_tensors <= kFewTensors ? run_clip<kFewTensors> : run_clip<kManyTensors>;
    const cudaError_t e = run(d_tensors, sizes, types, n_tensors, d_outs, max_norm, d_norm, (double*)d_workspace,
                              (cudaStream_t)stream);
    return e == cudaSuccess ? GAFIME_SUCCESS : status_from(e);
}
