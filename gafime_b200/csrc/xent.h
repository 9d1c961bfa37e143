// xent.h -- softmax cross entropy of a linear head: what its paths share.
//   xent.cu      entry points, argument checks, the choice of path, losses of a few rows
//   xent_few.cuh few classes: one pass over x (xent_few_*.cu: an instance a type)
//   xent_tc.cu   many classes: logits, gradients of x and w as tcgen05 products
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/gafime_b200.h"

namespace gafime {

// One call: z = x w^T + bias over n rows, d features and c classes; strides in elements.
struct XentCall {
    int type;                    // GAFIME_TYPE_*
    const void* x;
    int64_t xr, xk;              // strides of a row and of a feature
    const void* w;
    int64_t wr, wk;              // strides of a class and of a feature
    const float* bias;           // nullable, [c]
    const int64_t* labels;       // [n]; negative: the row is left out
    int64_t n, d, c;
    const float* weight;         // nullable, row weights of the gradient
    int64_t weight_stride;
    float scale;                 // times the row weight
    bool have_lse;               // loss and lse are inputs (a forward call wrote them)
    float* loss;                 // [n]
    float* lse;                  // [n]
    void* dx;                    // nullable
    int64_t dxr, dxk;
    void* dw;                    // nullable, [c][d]
    float* dbias;                // nullable, [c]
    bool gradient;               // a gradient call (dx, dw and dbias may still all be null)
    uint8_t* ws;
    size_t ws_bytes;
    cudaStream_t stream;
};

inline size_t xent_type_size(int type) { return type == GAFIME_TYPE_FP32 ? 4 : 2; }

// Hands out 256-byte aligned pieces of the workspace; with a null base it only counts them.
struct Carver {
    uint8_t* base;
    size_t used = 0;
    explicit Carver(uint8_t* b) : base(b) {}
    template <typename T>
    T* take(size_t count) {
        const size_t at = used;
        used += (count * sizeof(T) + 255) / 256 * 256;
        return base ? reinterpret_cast<T*>(base + at) : nullptr;
    }
};

// A kernel's dynamic shared memory, allowed once a device.  The limit belongs to the kernel, not to a
// launch: were it set to each call's own size, a smaller call of another thread could lower it
// between a call's setting and its launch.  One object for each kernel, always with the same size.
class SharedMemory {
public:
    cudaError_t allow(const void* kernel, size_t bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 64 && ((allowed_.load(std::memory_order_relaxed) >> dev) & 1)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess && dev < 64) allowed_.fetch_or(1ull << dev, std::memory_order_relaxed);
        return e;
    }

private:
    std::atomic<uint64_t> allowed_{0};
};

// Few classes: true when the class and feature counts fit its registers.
bool xent_few_fits(const XentCall& a);
size_t xent_few_workspace(const XentCall& a, int sms);
cudaError_t xent_few(const XentCall& a, int sms);

// Many classes (xent_tc.cu).
size_t xent_tc_workspace(const XentCall& a, int sms);
cudaError_t xent_tc(const XentCall& a, int sms);

// Packed pairs of floats: one instruction works on both (f32x2).
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ void unpair(float& lo, float& hi, Pair p) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
template <typename T>
__device__ __forceinline__ float to_float(T v) {
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace gafime
