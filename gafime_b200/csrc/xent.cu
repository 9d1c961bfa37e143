// xent.cu -- softmax cross entropy of a linear head: entry points and the few-class path.
//
//   z_ij = sum_k x_ik w_jk + b_j        lse_i = log sum_j exp z_ij      loss_i = lse_i - z_i,y(i)
//   g_ij = r_i (exp(z_ij - lse_i) - [j = y(i)])
//   dx = g w      dw = g^T x      dbias_j = sum_i g_ij
//
// Rows with a negative label are left out: loss and lse 0, no part in any gradient, whatever
// their features hold.  A label >= c makes the row's loss, and every gradient it enters, NaN.
//
// Few classes: xent_few.cuh.  Many: xent_tc.cu.  This file: the choice between them, the sum of
// the few-class path's partial gradients, argument checks and entry points.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "engine.h"
#include "xent.h"
#include "xent_few.cuh"

namespace gafime {

namespace {

constexpr int kFewMaxD = 2048;

// dw[c][k] = sum over p of part[p][c][k], and the bias's, fp64 in a fixed order.  A CTA adds
// eight neighbouring outputs (a sector of each partial): 128 threads share an output's partials,
// of which there are up to 24 an SM, so that two batches of loads read them (4e6 x 16 with 2
// classes: 9 us; 32 outputs a CTA, 19).
constexpr int kSumOut = 8;
template <typename T>
__global__ void __launch_bounds__(1024) xent_few_sum_kernel(const float* __restrict__ part,
                                                            const double* __restrict__ part_bias, int parts, int c, int d,
                                                            int d_pad, T* __restrict__ dw, float* __restrict__ dbias) {
    constexpr int kShare = 1024 / kSumOut;
    __shared__ double s[32][kSumOut + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int out = threadIdx.x % kSumOut, share = threadIdx.x / kSumOut;
    const int blocks_k = (d + kSumOut - 1) / kSumOut;
    const bool is_bias = !dw || (int)blockIdx.x >= c * blocks_k;
    const int cls = is_bias ? 0 : blockIdx.x / blocks_k, k = is_bias ? out : (blockIdx.x % blocks_k) * kSumOut + out;
    double v = 0.0;
    if (is_bias) {
        if (k < c)
            #pragma unroll 16
            for (int p = share; p < parts; p += kShare) v += part_bias[(size_t)p * c + k];
    } else if (k < d) {
        const float* q = part + (size_t)cls * d_pad + k;
        #pragma unroll 16
        for (int p = share; p < parts; p += kShare) v += (double)q[(size_t)p * c * d_pad];
    }
    #pragma unroll
    for (int o = 16; o >= kSumOut; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
    if (lane < kSumOut) s[warp][lane] = v;
    __syncthreads();
    if (warp >= kSumOut) return;
    // transposed: a warp adds one output's 32 sums
    v = s[lane][warp];
    #pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
    if (lane != 0) return;
    if (is_bias) {
        if (warp < c && dbias) dbias[warp] = (float)v;
    } else {
        const int ko = (blockIdx.x % blocks_k) * kSumOut + warp;
        if (ko < d) dw[(size_t)cls * d + ko] = from_float<T>((float)v);
    }
}
static_assert(kFewMaxGrad <= kSumOut, "the bias's sums are one CTA's");

// ---- a few rows, any number of classes ----------------------------------------------------
// Losses of up to kRowsFew rows (serving's single rows): bound by reading w once.  A warp takes
// classes in turn, its lanes the features, and keeps every row's running maximum and sum; the
// tensor cores would spend a tile of 256 rows on each class tile.  One row against 50000 x 1000 in
// bf16: 24 us (4,200 GB/s; 31 on the tensor cores' path with 128-row tiles, 42 with pairs).
constexpr int kRowsFew = 8;
constexpr int64_t kRowsFewValues = 12288;   // of x, fp32 in shared memory
constexpr size_t kRowsMaxSmem = 80 * 1024;   // eight rows' room for five of 2457 values, in whole units
constexpr int kRowsThreads = 256;
constexpr int rows_ctas(int64_t n) { return n <= 1 ? 3 : 2; }   // an SM holds, by registers

// 16 bytes of w, or one value where its rows are not made of them
template <typename T, bool VEC>
struct WLoad {
    static constexpr int kCount = VEC ? 16 / sizeof(T) : 1;
    static __device__ __forceinline__ void load(float (&v)[kCount], const T* p) {
        if constexpr (!VEC) {
            v[0] = to_float(*p);
        } else {
            const uint4 t = __ldg(reinterpret_cast<const uint4*>(p));
            if constexpr (sizeof(T) == 4) {
                v[0] = __uint_as_float(t.x);
                v[1] = __uint_as_float(t.y);
                v[2] = __uint_as_float(t.z);
                v[3] = __uint_as_float(t.w);
            } else {
                few::load4(reinterpret_cast<float(&)[4]>(v[0]), reinterpret_cast<const uint8_t*>(&t), T{});
                few::load4(reinterpret_cast<float(&)[4]>(v[4]), reinterpret_cast<const uint8_t*>(&t) + 8, T{});
            }
        }
    }
};

struct RowsArgs {
    const void* x;
    int64_t xr, xk;
    const void* w;
    int64_t wr, wk;
    const float* bias;
    const int64_t* labels;
    int n, d;
    int64_t c;
    float2* part;       // [n][warps of the grid]
    float* zy;          // [n], the label's logit
};

// N rows; x in shared memory as [units][N][values of a unit], zero past the features.  J classes
// at a time keep as many loads under way.
template <typename T, int N, bool VEC>
__global__ void __launch_bounds__(kRowsThreads, rows_ctas(N)) xent_rows_kernel(const RowsArgs a) {
    constexpr int V = WLoad<T, VEC>::kCount, J = N <= 2 ? 4 : N <= 4 ? 2 : 1;
    extern __shared__ __align__(16) float xs[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int units = (a.d + V - 1) / V, whole = a.d / V;
    for (int i = threadIdx.x; i < units * V * N; i += kRowsThreads) {
        const int v = i % V, r = i / V % N, k = i / (V * N) * V + v;
        xs[i] = r < a.n && k < a.d ? to_float(((const T*)a.x)[r * a.xr + k * a.xk]) : 0.f;
    }
    __syncthreads();
    float top[N], sum[N];
    int64_t y[N];
    #pragma unroll
    for (int r = 0; r < N; ++r) {
        top[r] = -INFINITY;
        sum[r] = 0.f;
        y[r] = r < a.n ? a.labels[r] : -1;
    }
    const int64_t first = (int64_t)blockIdx.x * (kRowsThreads / 32) + warp, step = (int64_t)gridDim.x * (kRowsThreads / 32);
    for (int64_t j0 = first * J; j0 < a.c; j0 += step * J) {
        const T* w[J];
        #pragma unroll
        for (int j = 0; j < J; ++j) w[j] = (const T*)a.w + min(j0 + j, a.c - 1) * a.wr;
        float z[J][N];
        #pragma unroll
        for (int j = 0; j < J; ++j)
            #pragma unroll
            for (int r = 0; r < N; ++r) z[j][r] = 0.f;
        #pragma unroll 2
        for (int q = lane; q < whole; q += 32) {
            float v[J][V];
            #pragma unroll
            for (int j = 0; j < J; ++j) WLoad<T, VEC>::load(v[j], w[j] + (int64_t)q * V * (VEC ? 1 : a.wk));
            #pragma unroll
            for (int r = 0; r < N; ++r)
                #pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xv = xs[(q * N + r) * V + i];
                    #pragma unroll
                    for (int j = 0; j < J; ++j) z[j][r] = fmaf(v[j][i], xv, z[j][r]);
                }
        }
        if (VEC && whole * V + lane < a.d) {   // the features past the last unit
            #pragma unroll
            for (int j = 0; j < J; ++j) {
                const float v = to_float(w[j][whole * V + lane]);
                #pragma unroll
                for (int r = 0; r < N; ++r) z[j][r] = fmaf(v, xs[(whole * N + r) * V + lane], z[j][r]);
            }
        }
        #pragma unroll
        for (int o = 16; o; o >>= 1)
            #pragma unroll
            for (int j = 0; j < J; ++j)
                #pragma unroll
                for (int r = 0; r < N; ++r) z[j][r] += __shfl_xor_sync(0xffffffffu, z[j][r], o);
        #pragma unroll
        for (int j = 0; j < J; ++j) {
            if (j0 + j >= a.c) break;
            const float b = a.bias ? a.bias[j0 + j] : 0.f;
            #pragma unroll
            for (int r = 0; r < N; ++r) {
                const float v = z[j][r] + b, m = fmaxf(top[r], v), shift = m == -INFINITY ? 0.f : m;
                sum[r] = sum[r] * expf(top[r] - shift) + expf(v - shift);
                top[r] = m;
                if (j0 + j == y[r] && lane == 0) a.zy[r] = v;
            }
        }
    }
    if (lane == 0)
        #pragma unroll
        for (int r = 0; r < N; ++r)
            if (r < a.n) a.part[r * step + first] = make_float2(top[r], sum[r]);
}

// a block a row: loss and lse from the warps' maxima and sums, in a fixed order
__global__ void __launch_bounds__(256) xent_rows_join_kernel(const float2* __restrict__ part, int64_t parts, int64_t c,
                                                             const float* __restrict__ zy,
                                                             const int64_t* __restrict__ labels, float* loss, float* lse) {
    __shared__ float s[8];
    const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float2* p = part + r * parts;
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < parts; i += 256) m = fmaxf(m, p[i].x);
    #pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s[warp] = m;
    __syncthreads();
    for (int i = 0; i < 8; ++i) m = fmaxf(m, s[i]);
    if (m == -INFINITY) m = 0.f;
    float t = 0.f;
    for (int64_t i = threadIdx.x; i < parts; i += 256) t += p[i].y * expf(p[i].x - m);
    #pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    __syncthreads();
    if (lane == 0) s[warp] = t;
    __syncthreads();
    if (threadIdx.x != 0) return;
    t = 0.f;
    for (int i = 0; i < 8; ++i) t += s[i];
    const int64_t y = labels[r];
    const float l = logf(t);
    loss[r] = y < 0 ? 0.f : y < c ? (m - zy[r]) + l : NAN;
    if (lse) lse[r] = y < 0 ? 0.f : m + l;
}

bool rows_fit(const XentCall& a) {
    return !a.gradient && a.n >= 1 && a.n <= kRowsFew && a.n * a.d <= kRowsFewValues && a.c >= 32;
}
int rows_grid(const XentCall& a, int sms) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)rows_ctas(a.n) * sms, (a.c + 8 * 4 - 1) / (8 * 4)));   // four classes a warp
}
size_t rows_carve(const XentCall& a, int sms, uint8_t* ws, float2*& part, float*& zy) {
    Carver cv(ws);
    part = cv.take<float2>((size_t)a.n * rows_grid(a, sms) * (kRowsThreads / 32));
    zy = cv.take<float>(a.n);
    return cv.used;
}
template <typename T, int N, bool VEC>
cudaError_t rows_launch_as(const RowsArgs& r, int grid, cudaStream_t st) {
    constexpr int V = WLoad<T, VEC>::kCount;
    const size_t smem = (size_t)((r.d + V - 1) / V) * V * N * sizeof(float);
    auto fn = xent_rows_kernel<T, N, VEC>;
    static SharedMemory shared;
    const cudaError_t e = shared.allow((const void*)fn, kRowsMaxSmem);
    if (e != cudaSuccess) return e;
    KernelTimer kt(st, GAFIME_KERNEL_XENT);
    fn<<<grid, kRowsThreads, smem, st>>>(r);
    return cudaGetLastError();
}
template <typename T, int N>
cudaError_t rows_launch(const RowsArgs& r, int grid, cudaStream_t st) {
    const bool vec = r.wk == 1 && (uintptr_t)r.w % 16 == 0 && r.wr * (int64_t)sizeof(T) % 16 == 0;
    return vec ? rows_launch_as<T, N, true>(r, grid, st) : rows_launch_as<T, N, false>(r, grid, st);
}
template <typename T>
cudaError_t rows_run(const XentCall& a, int sms) {
    RowsArgs r{};
    r.x = a.x; r.xr = a.xr; r.xk = a.xk; r.w = a.w; r.wr = a.wr; r.wk = a.wk;
    r.bias = a.bias; r.labels = a.labels; r.n = (int)a.n; r.d = (int)a.d; r.c = a.c;
    rows_carve(a, sms, a.ws, r.part, r.zy);
    const int grid = rows_grid(a, sms);
    cudaError_t e = a.n == 1   ? rows_launch<T, 1>(r, grid, a.stream)
                    : a.n == 2 ? rows_launch<T, 2>(r, grid, a.stream)
                    : a.n <= 4 ? rows_launch<T, 4>(r, grid, a.stream)
                               : rows_launch<T, 8>(r, grid, a.stream);
    if (e != cudaSuccess) return e;
    KernelTimer kt(a.stream, GAFIME_KERNEL_XENT);
    xent_rows_join_kernel<<<(unsigned)a.n, 256, 0, a.stream>>>(r.part, (int64_t)grid * (kRowsThreads / 32), a.c, r.zy,
                                                               a.labels, a.loss, a.lse);
    return cudaGetLastError();
}

FewPlan few_plan(const XentCall& a, int sms) {
    FewPlan p{};
    const int d = (int)a.d, c = (int)a.c, es = (int)xent_type_size(a.type);
    p.cp = c <= 4 ? std::max(2, c) : c <= 6 ? 6 : c <= 8 ? 8 : 16;
    const int line = (p.cp + 1) / 2 * 2;   // classes of a line of w and g in shared memory
    p.cols = a.xr == 1 && a.xk != 1;
    p.grad = a.gradient && (a.dw || a.dbias || a.dx);
    FewArgs& k = p.k;
    k.x = a.x; k.xr = a.xr; k.xk = a.xk; k.w = a.w; k.wr = a.wr; k.wk = a.wk;
    k.bias = a.bias; k.labels = a.labels; k.n = a.n; k.d = d; k.c = c;
    k.weight = a.weight; k.weight_stride = a.weight_stride; k.scale = a.scale;
    k.have_lse = a.have_lse;
    k.loss = a.loss; k.lse = a.lse; k.dx = a.dx; k.dxr = a.dxr; k.dxk = a.dxk;
    p.features = few_features(p.grad, d <= 64);
    k.d_pad = (d + p.features - 1) / p.features * p.features;
    const int64_t line_stride = p.cols ? a.xk : a.xr;
    p.vec = (p.cols ? a.xr == 1 : a.xk == 1) && (uintptr_t)a.x % 16 == 0 && line_stride >= 0 &&
               line_stride * es % 16 == 0;
    k.warps = p.grad ? k.d_pad / p.features : 1;
    k.groups = std::max(1, (p.grad ? 4 : 8) / k.warps);
    const int warps = k.warps * k.groups;
    p.threads = 32 * warps;
    auto smem = [&](int rows) {
        return (size_t)warps * rows * p.features * es +
               sizeof(float) * ((size_t)k.d_pad * line + (p.grad ? (size_t)warps * kRowsMost * line * (p.cols ? 1 : 2) : 0) +
                                (p.grad && k.warps > 1 ? 2 * (size_t)warps * p.cp * 32 : 0)) +
               (p.grad ? sizeof(double) * k.groups * p.cp * 32 : 0);
    };
    // CTAs an SM holds
    auto resident = [&](int rows) {
        return (int)std::min<size_t>(few_warps(p.cp, p.features, p.grad) / warps, (227 * 1024) / (smem(rows) + 1024));
    };
    // Rows of a tile: 32, half of that where fewer than ten warps an SM would be left, and fewer
    // still where SMs would be left without a tile
    int rows = kRowsMost;
    if (resident(rows) * warps < 10 && resident(16) * warps > resident(rows) * warps) rows = 16;
    while (rows > 8 && ((a.n + rows - 1) / rows < 4 * sms || resident(rows) < 1)) rows /= 2;
    // By columns the tiles of a CTA's groups (without gradients, of two sets of them) lie side by
    // side: longer pieces of a column
    p.beside = 1;
    if (p.cols && p.vec && rows == 32) {
        if (!p.grad && p.cp <= kBesideMaxC && d >= kBesideMinD) p.beside = 4;
        if (p.grad && (k.groups == 4 || k.groups == 2)) p.beside = k.groups;
    }
    k.rows = rows;
    k.log_rows = rows == 32 ? 5 : rows == 16 ? 4 : 3;
    k.n_tiles = (int)((a.n + rows - 1) / rows);
    p.smem = smem(rows);
    p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(k.n_tiles, (int64_t)std::max(1, resident(rows)) * sms));
    return p;
}

size_t few_carve(const XentCall& a, FewPlan& p, uint8_t* ws) {
    Carver cv(ws);
    if (p.grad) {
        const size_t parts = (size_t)p.grid * p.k.groups;
        p.k.part = a.dw ? cv.take<float>(parts * a.c * p.k.d_pad) : nullptr;
        p.k.part_bias = cv.take<double>(parts * a.c);
    }
    return cv.used;
}

template <typename T>
cudaError_t few_sum(const XentCall& a, const FewPlan& p) {
    const int blocks = (a.dw ? (int)a.c * (((int)a.d + kSumOut - 1) / kSumOut) : 0) + (a.dbias ? 1 : 0);
    KernelTimer kt(a.stream, GAFIME_KERNEL_XENT);
    xent_few_sum_kernel<T><<<blocks, 1024, 0, a.stream>>>(p.k.part, p.k.part_bias, a.n > 0 ? p.grid * p.k.groups : 0,
                                                          (int)a.c, (int)a.d, p.k.d_pad, (T*)a.dw, a.dbias);
    return cudaGetLastError();
}

}  // namespace

bool xent_few_fits(const XentCall& a) {
    if (a.c > kFewMaxC || a.d > kFewMaxD) return false;
    if (a.gradient && (a.dx || a.dw || a.dbias) && a.c > kFewMaxGrad) return false;
    const FewPlan p = few_plan(a, 148);
    return p.threads <= 512 && p.smem <= kFewMaxSmem;
}

size_t xent_few_workspace(const XentCall& a, int sms) {
    FewPlan p = few_plan(a, sms);
    return few_carve(a, p, nullptr);
}

template <typename T>
static cudaError_t few_run(const XentCall& a, const FewPlan& p) {
    if (a.n > 0) {
        const cudaError_t e = p.cols ? few_launch_columns(p, a.stream, T{}) : few_launch_rows(p, a.stream, T{});
        if (e != cudaSuccess) return e;
    }
    return p.grad && (a.dw || a.dbias) ? few_sum<T>(a, p) : cudaSuccess;
}

cudaError_t xent_few(const XentCall& a, int sms) {
    FewPlan p = few_plan(a, sms);
    few_carve(a, p, a.ws);
    switch (a.type) {
        case GAFIME_TYPE_FP32: return few_run<float>(a, p);
        case GAFIME_TYPE_FP16: return few_run<__half>(a, p);
        default: return few_run<__nv_bfloat16>(a, p);
    }
}

// ---- entry points ---------------------------------------------------------------------

namespace {

int sm_count_of_current() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

bool sizes_ok(int type, int64_t n, int64_t d, int64_t c) {
    return (type == GAFIME_TYPE_FP32 || type == GAFIME_TYPE_FP16 || type == GAFIME_TYPE_BF16) && n >= 0 && d >= 1 &&
           c >= 1 && n <= 0x7fffff00ll && d <= 0x7fffff00ll && c <= 0x7fffff00ll;
}

bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

// Pointers on their elements' boundaries, and strides that the kernels can follow.
bool layout_ok(const XentCall& a) {
    const size_t es = xent_type_size(a.type);
    if (!aligned(a.x, es) || !aligned(a.w, es) || !aligned(a.dx, es) || !aligned(a.dw, es) || !aligned(a.labels, 8) ||
        !aligned(a.bias, 4) || !aligned(a.weight, 4) || !aligned(a.loss, 4) || !aligned(a.lse, 4) || !aligned(a.dbias, 4))
        return false;
    if (a.xr < 0 || a.xk < 0 || a.wr < 0 || a.wk < 0 || a.weight_stride < 0 || a.dxr < 0 || a.dxk < 0) return false;
    // every element of dx has a place of its own
    return !a.dx || ((a.n <= 1 || a.dxr > 0) && (a.d <= 1 || a.dxk > 0) && (a.n <= 1 || a.d <= 1 || a.dxr != a.dxk));
}

size_t workspace_of(const XentCall& a) {
    const int sms = sm_count_of_current();
    if (rows_fit(a)) {
        float2* part;
        float* zy;
        return rows_carve(a, sms, nullptr, part, zy);
    }
    return xent_few_fits(a) ? xent_few_workspace(a, sms) : xent_tc_workspace(a, sms);
}

int run_xent(const XentCall& a) {
    if (!layout_ok(a)) return GAFIME_ERROR_INVALID_ARGS;
    if (gafime_cuda_available() != 1) return GAFIME_ERROR_CUDA_NOT_AVAILABLE;
    if (a.n == 0 && !a.dw && !a.dbias) return GAFIME_SUCCESS;
    const size_t need = workspace_of(a);
    if (need > a.ws_bytes || (need && (!a.ws || (uintptr_t)a.ws % 256))) return GAFIME_ERROR_INVALID_ARGS;
    const int sms = sm_count_of_current();
    cudaError_t e;
    if (rows_fit(a))
        e = a.type == GAFIME_TYPE_FP32   ? rows_run<float>(a, sms)
            : a.type == GAFIME_TYPE_FP16 ? rows_run<__half>(a, sms)
                                         : rows_run<__nv_bfloat16>(a, sms);
    else
        e = xent_few_fits(a) ? xent_few(a, sms) : xent_tc(a, sms);
    return e == cudaSuccess ? GAFIME_SUCCESS : status_from(e);
}

}  // namespace

}  // namespace gafime

using namespace gafime;

extern "C" int gafime_xent_workspace(int type, const void* d_x, int64_t x_row, int64_t x_col, const void* d_w,
                                     int64_t w_row, int64_t w_col, int64_t n, int64_t d, int64_t c, int want,
                                     size_t* bytes_out) {
    if (!bytes_out || !sizes_ok(type, n, d, c) || want < 0 || want > 15) return GAFIME_ERROR_INVALID_ARGS;
    XentCall a{};
    a.type = type;
    a.x = d_x; a.xr = x_row; a.xk = x_col;
    a.w = d_w; a.wr = w_row; a.wk = w_col;
    a.n = n; a.d = d; a.c = c;
    a.gradient = want != 0;
    // only their being there matters to the plan
    a.dx = want & GAFIME_XENT_DX ? (void*)1 : nullptr;
    a.dw = want & GAFIME_XENT_DW ? (void*)1 : nullptr;
    a.dbias = want & GAFIME_XENT_DBIAS ? (float*)4 : nullptr;
    *bytes_out = workspace_of(a);
    return GAFIME_SUCCESS;
}

extern "C" int gafime_xent_forward(int type, const void* d_x, int64_t x_row, int64_t x_col, const void* d_w,
                                   int64_t w_row, int64_t w_col, const float* d_bias, const int64_t* d_labels,
                                   int64_t n, int64_t d, int64_t c, float* d_loss, float* d_lse, void* d_workspace,
                                   size_t workspace_bytes, void* stream) {
    if (!sizes_ok(type, n, d, c) || !d_w || (n > 0 && (!d_x || !d_labels || !d_loss)))
        return GAFIME_ERROR_INVALID_ARGS;
    XentCall a{};
    a.type = type;
    a.x = d_x; a.xr = x_row; a.xk = x_col;
    a.w = d_w; a.wr = w_row; a.wk = w_col;
    a.bias = d_bias; a.labels = d_labels;
    a.n = n; a.d = d; a.c = c;
    a.loss = d_loss; a.lse = d_lse;
    a.ws = (uint8_t*)d_workspace; a.ws_bytes = workspace_bytes;
    a.stream = (cudaStream_t)stream;
    return run_xent(a);
}

extern "C" int gafime_xent_gradient(int type, const void* d_x, int64_t x_row, int64_t x_col, const void* d_w,
                                    int64_t w_row, int64_t w_col, const float* d_bias, const int64_t* d_labels,
                                    int64_t n, int64_t d, int64_t c, const float* d_row_weight,
                                    int64_t row_weight_stride, float scale, int have_lse, float* d_loss,
                                    float* d_lse, void* d_dx, int64_t dx_row, int64_t dx_col, void* d_dw,
                                    float* d_dbias, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (!sizes_ok(type, n, d, c) || !d_w || (n > 0 && (!d_x || !d_labels || !d_loss)) || (have_lse && n > 0 && !d_lse))
        return GAFIME_ERROR_INVALID_ARGS;
    XentCall a{};
    a.type = type;
    a.x = d_x; a.xr = x_row; a.xk = x_col;
    a.w = d_w; a.wr = w_row; a.wk = w_col;
    a.bias = d_bias; a.labels = d_labels;
    a.n = n; a.d = d; a.c = c;
    a.weight = d_row_weight; a.weight_stride = row_weight_stride; a.scale = scale;
    a.have_lse = have_lse != 0;
    a.loss = d_loss; a.lse = d_lse;
    a.dx = d_dx; a.dxr = dx_row; a.dxk = dx_col;
    a.dw = d_dw; a.dbias = d_dbias;
    a.gradient = true;
    a.ws = (uint8_t*)d_workspace; a.ws_bytes = workspace_bytes;
    a.stream = (cudaStream_t)stream;
    return run_xent(a);
}
