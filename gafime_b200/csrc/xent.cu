// xent.cu -- softmax cross entropy of a linear head: entry points and the few-class path.
//
//   z_ij = sum_k x_ik w_jk + b_j        lse_i = log sum_j exp z_ij      loss_i = lse_i - z_i,y(i)
//   g_ij = r_i (exp(z_ij - lse_i) - [j = y(i)])
//   dx = g w      dw = g^T x      dbias_j = sum_i g_ij
//
// Rows with a negative label are left out: loss and lse 0, no part in any gradient, whatever
// their features hold.  A label >= c makes the row's loss, and every gradient it enters, NaN.
//
// Few classes (this file): every logit of a row fits into registers, so one pass over x gives
// the loss and the gradient of w; nothing of size n x c exists.  The pass is bound by reading
// x.  A CTA walks over tiles of rows held in shared memory (the next tile's cp.async copies in
// flight meanwhile):
//   1. a thread is one row and one slice of the features: c partial dot products; slices are
//      added through shared memory
//   2. one thread a row: softmax, loss, and the row's g to shared memory
//   3. a thread is one or more features: c sums of g x over the tile's rows, added to running
//      sums at the tile's end (two short fp32 chains in place of one long one)
// and leaves its sums of w's gradient to xent_few_sum_kernel, which adds them in fp64 in a
// fixed order.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "engine.h"
#include "xent.h"

namespace gafime {

namespace {

constexpr int kFewThreads = 256;
constexpr int kFewTileBytes = 40 * 1024;  // of x; two tiles a CTA, two CTAs an SM
constexpr int kFewMaxC = 16;
constexpr int kFewMaxD = 2048;
constexpr int kFewMaxRows = 256;
constexpr size_t kFewMaxSmem = 226 * 1024;

struct FewArgs {
    const void* x;
    int64_t xr, xk;
    const void* w;
    int64_t wr, wk;
    const float* bias;
    const int64_t* labels;
    int64_t n;
    int d, c;
    const float* weight;
    int64_t weight_stride;
    float scale;
    int have_lse, want_dw;
    float* loss;
    float* lse;
    void* dx;
    int64_t dxr, dxk;
    float* part;        // [grid][row slices][c][d], then [grid][c] of the bias
    float* part_bias;
    int rows;           // rows of a tile, a power of two
    int log_rows;
    int pitch;          // elements between the tile's rows (columns: features) in shared memory
    int vec_ok;         // 16-byte copies allowed
    int stages;         // tiles held at a time: 2, or 1 where only one fits
    int log_dc;         // log2 of the threads along the features in step 3
    int n_tiles;
};

template <typename T>
__device__ __forceinline__ void cp_async16(uint32_t dst, const T* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Queue the copies of tile t: rows [t R, t R + R) of x; what lies past the table reads zero.
template <typename T, bool COLS>
__device__ __forceinline__ void few_load(const FewArgs& a, T* tile, int t, int tid) {
    constexpr int V = 16 / sizeof(T);
    const int R = a.rows;
    const int64_t r0 = (int64_t)t * R;
    const int left = (int)min((int64_t)R, a.n - r0);
    const T* x = (const T*)a.x + r0 * a.xr;
    if (a.vec_ok) {
        const uint32_t dst0 = (uint32_t)__cvta_generic_to_shared(tile);
        const int lines = COLS ? a.d : R;            // contiguous runs of the tile
        const int len = COLS ? left : a.d;           // elements of a run
        const int nv = ((COLS ? R : a.d) + V - 1) / V;
        const int valid = COLS ? a.d : left;
        const int64_t ls = COLS ? a.xk : a.xr;
        // copy i is vector i % nv of line i / nv; the line advances without a division per copy
        int line = tid / nv, v = tid - line * nv;
        const int dl = kFewThreads / nv, dv = kFewThreads - dl * nv;
        while (line < lines) {
            const int left_v = min(V, len - v * V);
            const int bytes = line < valid && left_v > 0 ? left_v * (int)sizeof(T) : 0;
            const T* src = bytes ? x + line * ls + v * V : x;
            cp_async16(dst0 + (uint32_t)((line * a.pitch + v * V) * (int)sizeof(T)), src, bytes);
            line += dl;
            v += dv;
            if (v >= nv) {
                v -= nv;
                ++line;
            }
        }
    } else {
        // any strides: element by element, neighbouring threads on neighbouring addresses
        const int inner = COLS ? R : (a.d + V - 1) / V * V, lines = COLS ? a.d : R;
        int line = tid / inner, e = tid - line * inner;
        const int dl = kFewThreads / inner, de = kFewThreads - dl * inner;
        while (line < lines) {
            const int r = COLS ? e : line, k = COLS ? line : e;
            tile[line * a.pitch + e] = r < left && k < a.d ? x[r * a.xr + k * a.xk] : from_float<T>(0.f);
            line += dl;
            e += de;
            if (e >= inner) {
                e -= inner;
                ++line;
            }
        }
    }
}

template <int CP>
__device__ __forceinline__ void load_vec(float (&v)[CP], const float* p) {
    if constexpr (CP == 2) {
        const float2 t = *reinterpret_cast<const float2*>(p);
        v[0] = t.x;
        v[1] = t.y;
    } else {
        #pragma unroll
        for (int c = 0; c < CP; c += 4) {
            const float4 t = *reinterpret_cast<const float4*>(p + c);
            v[c] = t.x;
            v[c + 1] = t.y;
            v[c + 2] = t.z;
            v[c + 3] = t.w;
        }
    }
}

// 16 bytes of a line as floats
__device__ __forceinline__ void load_line(float (&v)[4], const float* p) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x;
    v[1] = t.y;
    v[2] = t.z;
    v[3] = t.w;
}
__device__ __forceinline__ void load_line(float (&v)[8], const __half* p) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {t.x, t.y, t.z, t.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load_line(float (&v)[8], const __nv_bfloat16* p) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {t.x, t.y, t.z, t.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

// CP: classes padded to 2, 4, 8 or 16; KPT: features a thread owns in step 3 (0: no gradient)
template <typename T, int CP, int KPT, bool COLS>
__global__ void __launch_bounds__(kFewThreads, (CP * (KPT ? KPT : 1) <= 16 ? 2 : 1)) xent_few_kernel(FewArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int R = a.rows, d = a.d;
    const int tile_elems = (COLS ? d : R) * a.pitch;
    const size_t tile_bytes = ((size_t)tile_elems * sizeof(T) + 127) / 128 * 128;
    float* ws = reinterpret_cast<float*>(smem + a.stages * tile_bytes);   // w: [d][CP], whole vectors
    constexpr int V = 16 / sizeof(T);
    const int dv = (d + V - 1) / V * V;
    float* gs = ws + (size_t)dv * CP;                              // g: [R][CP]
    const int slots = R >= 32 ? kFewThreads / R : kFewThreads / 32;
    float* red = gs + R * CP;                                      // [slots][R][CP]
    float* bs = red + slots * R * CP;                              // bias [CP]
    uint32_t* keep = reinterpret_cast<uint32_t*>(bs + CP);         // rows that count, 32 a word

    for (int i = tid; i < dv * CP; i += kFewThreads) {
        const int k = i / CP, c = i % CP;
        ws[i] = c < a.c && k < d ? to_float(((const T*)a.w)[c * a.wr + k * a.wk]) : 0.f;
    }
    if (tid < CP) bs[tid] = tid < a.c ? (a.bias ? a.bias[tid] : 0.f) : -INFINITY;

    constexpr int KP = KPT ? KPT : 1;
    float sum[KP][CP];
    double dbias[CP];
    #pragma unroll
    for (int j = 0; j < KP; ++j)
        #pragma unroll
        for (int c = 0; c < CP; ++c) sum[j][c] = 0.f;
    #pragma unroll
    for (int c = 0; c < CP; ++c) dbias[c] = 0.0;

    const int row = tid & (R - 1), slice = tid >> a.log_rows, n_slices = kFewThreads >> a.log_rows;
    const int dc = 1 << a.log_dc;                       // threads along the features
    const int k0 = tid & (dc - 1), rs = tid >> a.log_dc, n_rs = kFewThreads >> a.log_dc;

    int t = blockIdx.x;
    if (t < a.n_tiles && a.stages == 2) few_load<T, COLS>(a, reinterpret_cast<T*>(smem), t, tid);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int it = 0; t < a.n_tiles; ++it, t += gridDim.x) {
        T* tile = reinterpret_cast<T*>(smem + (a.stages == 2 ? (it & 1) * tile_bytes : 0));
        if (a.stages == 2) {
            if (t + (int)gridDim.x < a.n_tiles)
                few_load<T, COLS>(a, reinterpret_cast<T*>(smem + ((it + 1) & 1) * tile_bytes), t + gridDim.x, tid);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            few_load<T, COLS>(a, tile, t, tid);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        // the label and weight of the row this thread will finish, early
        const int64_t gr = (int64_t)t * R + tid;
        int64_t y = -1;
        float rw = 0.f;
        if (tid < R && gr < a.n) {
            y = a.labels[gr];
            if (KPT || a.dx) rw = (a.weight ? a.weight[gr * a.weight_stride] : 1.f) * a.scale;
        }
        __syncthreads();

        // 1. partial logits
        {
            float z[CP];
            #pragma unroll
            for (int c = 0; c < CP; ++c) z[c] = 0.f;
            if (COLS) {
                for (int k = slice; k < d; k += n_slices) {
                    const float xv = to_float(tile[k * a.pitch + row]);
                    float wv[CP];
                    load_vec<CP>(wv, ws + k * CP);
                    #pragma unroll
                    for (int c = 0; c < CP; ++c) z[c] = fmaf(xv, wv[c], z[c]);
                }
            } else {
                for (int k = slice * V; k < d; k += n_slices * V) {
                    float xv[V];
                    load_line(xv, tile + row * a.pitch + k);
                    #pragma unroll
                    for (int v = 0; v < V; ++v) {
                        float wv[CP];
                        load_vec<CP>(wv, ws + (k + v) * CP);
                        #pragma unroll
                        for (int c = 0; c < CP; ++c) z[c] = fmaf(xv[v], wv[c], z[c]);
                    }
                }
            }
            // rows of fewer than 32 lanes: several slices share a warp
            for (int o = R; o < 32; o <<= 1)
                #pragma unroll
                for (int c = 0; c < CP; ++c) z[c] += __shfl_xor_sync(0xffffffffu, z[c], o);
            if (R >= 32 || lane < R) {
                float* p = red + ((R >= 32 ? slice : warp) * R + row) * CP;
                #pragma unroll
                for (int c = 0; c < CP; ++c) p[c] = z[c];
            }
        }
        __syncthreads();

        // 2. one thread a row
        if (tid < R) {
            float z[CP], v[CP];
            load_vec<CP>(z, bs);
            for (int s = 0; s < slots; ++s) {
                load_vec<CP>(v, red + (s * R + tid) * CP);
                #pragma unroll
                for (int c = 0; c < CP; ++c) z[c] += v[c];
            }
            float m = z[0];
            #pragma unroll
            for (int c = 1; c < CP; ++c) m = fmaxf(m, z[c]);
            if (m == -INFINITY) m = 0.f;   // every class excluded: exp(-inf) = 0, not NaN
            float s = 0.f, zy = NAN;       // a label >= c leaves NaN
            #pragma unroll
            for (int c = 0; c < CP; ++c) {
                s += expf(z[c] - m);
                if (y == c && c < a.c) zy = z[c];
            }
            const float ls = logf(s);
            const bool kept = y >= 0;
            float shift = m + ls;
            if (a.have_lse && gr < a.n) {
                shift = a.lse[gr];
            } else if (gr < a.n) {
                a.loss[gr] = kept ? (m - zy) + ls : 0.f;
                if (a.lse) a.lse[gr] = kept ? shift : 0.f;
            }
            if (KPT || a.dx) {
                const bool bad = kept && y >= a.c;
                #pragma unroll
                for (int c = 0; c < CP; ++c) {
                    // with this call's own sum the shift is taken in two steps: z - m is exact
                    // where it matters and log s is small
                    const float p = a.have_lse ? expf(z[c] - shift) : expf((z[c] - m) - ls);
                    float g = kept ? (p - (y == c ? 1.f : 0.f)) * rw : 0.f;
                    if (bad) g = NAN;
                    if (c >= a.c) g = 0.f;
                    gs[tid * CP + c] = g;
                    dbias[c] += g;
                }
                const uint32_t b = __ballot_sync(R >= 32 ? 0xffffffffu : (1u << R) - 1, kept);
                if (lane == 0) keep[tid >> 5] = b;
            }
        }
        if (KPT || a.dx) {
            __syncthreads();
            // 3. gradient of w: sums over the tile's rows, one or more features a thread
            if (KPT) {
                float acc[KP][CP];
                #pragma unroll
                for (int j = 0; j < KP; ++j)
                    #pragma unroll
                    for (int c = 0; c < CP; ++c) acc[j][c] = 0.f;
                if (COLS) {
                    for (int r = rs * V; r < R; r += n_rs * V) {
                        const uint32_t kept = (keep[r >> 5] >> (r & 31)) & ((1u << V) - 1);
                        if (!kept) continue;   // uniform in the warp, as all of `kept` is
                        float xv[KP][V];
                        #pragma unroll
                        for (int j = 0; j < KP; ++j) {
                            const int k = k0 + j * kFewThreads;
                            if (k < d) {
                                load_line(xv[j], tile + k * a.pitch + r);
                            } else {
                                #pragma unroll
                                for (int v = 0; v < V; ++v) xv[j][v] = 0.f;
                            }
                        }
                        #pragma unroll
                        for (int v = 0; v < V; ++v) {
                            if (!((kept >> v) & 1)) continue;
                            float g[CP];
                            load_vec<CP>(g, gs + (r + v) * CP);
                            #pragma unroll
                            for (int j = 0; j < KP; ++j)
                                #pragma unroll
                                for (int c = 0; c < CP; ++c) acc[j][c] = fmaf(g[c], xv[j][v], acc[j][c]);
                        }
                    }
                } else {
                    for (int r = rs; r < R; r += n_rs) {
                        if (!((keep[r >> 5] >> (r & 31)) & 1)) continue;   // uniform in the warp
                        float g[CP];
                        load_vec<CP>(g, gs + r * CP);
                        #pragma unroll
                        for (int j = 0; j < KP; ++j) {
                            const int k = k0 + j * kFewThreads;
                            if (k < d) {
                                const float xv = to_float(tile[r * a.pitch + k]);
                                #pragma unroll
                                for (int c = 0; c < CP; ++c) acc[j][c] = fmaf(g[c], xv, acc[j][c]);
                            }
                        }
                    }
                }
                #pragma unroll
                for (int j = 0; j < KP; ++j)
                    #pragma unroll
                    for (int c = 0; c < CP; ++c) sum[j][c] += acc[j][c];
            }
            // gradient of x
            if (a.dx) {
                const int64_t r0 = (int64_t)t * R;
                const int left = (int)min((int64_t)R, a.n - r0);
                T* dx = (T*)a.dx + r0 * a.dxr;
                if (COLS) {
                    // neighbouring threads are neighbouring rows
                    float g[CP];
                    load_vec<CP>(g, gs + row * CP);
                    if (row < left)
                        for (int k = slice; k < d; k += n_slices) {
                            float wv[CP], s = 0.f;
                            load_vec<CP>(wv, ws + k * CP);
                            #pragma unroll
                            for (int c = 0; c < CP; ++c) s = fmaf(g[c], wv[c], s);
                            dx[row * a.dxr + k * a.dxk] =
                                from_float<T>((keep[row >> 5] >> (row & 31)) & 1 ? s : 0.f);
                        }
                } else {
                    for (int k = tid & (dc - 1); k < d; k += dc) {
                        float wv[CP];
                        load_vec<CP>(wv, ws + k * CP);
                        for (int r = rs; r < left; r += n_rs) {
                            float g[CP], s = 0.f;
                            load_vec<CP>(g, gs + r * CP);
                            #pragma unroll
                            for (int c = 0; c < CP; ++c) s = fmaf(g[c], wv[c], s);
                            dx[r * a.dxr + k * a.dxk] = from_float<T>((keep[r >> 5] >> (r & 31)) & 1 ? s : 0.f);
                        }
                    }
                }
            }
        }
        __syncthreads();   // before the next copies overwrite this tile, and its g
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    if (KPT) {
        float* part = a.part + ((size_t)blockIdx.x * n_rs + rs) * a.c * d;
        #pragma unroll
        for (int j = 0; j < KP; ++j) {
            const int k = k0 + j * kFewThreads;
            if (k < d && a.want_dw)
                #pragma unroll
                for (int c = 0; c < CP; ++c)
                    if (c < a.c) part[(size_t)c * d + k] = sum[j][c];
        }
        // the bias: rows' sums through shared memory, in a fixed order
        __syncthreads();
        if (tid < R)
            #pragma unroll
            for (int c = 0; c < CP; ++c) gs[tid * CP + c] = (float)dbias[c];
        __syncthreads();
        if (tid < a.c) {
            double s = 0.0;
            for (int r = 0; r < R; ++r) s += gs[r * CP + tid];
            a.part_bias[(size_t)blockIdx.x * a.c + tid] = (float)s;
        }
    }
}

// out[e] = sum over p of part[p][e], fp64 in a fixed order: 16 warps split the partials of 32
// neighbouring outputs
template <typename T>
__global__ void __launch_bounds__(512) xent_few_sum_kernel(const float* __restrict__ part, int n_part, int64_t size,
                                                           T* __restrict__ out,
                                                           const float* __restrict__ part_bias, int n_bias, int c,
                                                           float* __restrict__ dbias) {
    __shared__ double s[16][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t blocks_w = out ? (size + 31) / 32 : 0;
    const bool is_bias = blockIdx.x >= blocks_w;
    const float* src = is_bias ? part_bias : part;
    const int64_t len = is_bias ? c : size;
    const int count = is_bias ? n_bias : n_part;
    const int64_t e = (is_bias ? (int64_t)blockIdx.x - blocks_w : (int64_t)blockIdx.x) * 32 + lane;
    double v = 0.0;
    if (e < len) {
        #pragma unroll 8
        for (int p = warp; p < count; p += 16) v += (double)src[(int64_t)p * len + e];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && e < len) {
        double tot = 0.0;
        #pragma unroll
        for (int i = 0; i < 16; ++i) tot += s[i][lane];
        if (is_bias)
            dbias[e] = (float)tot;
        else
            out[e] = from_float<T>((float)tot);
    }
}

struct FewPlan {
    FewArgs k;
    int cp, kpt, grid, n_rs;
    bool cols;
    size_t smem;
};

int pow2_ceil(int v) {
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}
int ilog2(int v) {
    int l = 0;
    while ((1 << l) < v) ++l;
    return l;
}

FewPlan few_plan(const XentCall& a, int sms) {
    FewPlan p{};
    const int d = (int)a.d, es = (int)xent_type_size(a.type), V = 16 / es;
    p.cp = std::max(2, pow2_ceil((int)a.c));
    p.cols = a.xr == 1 && a.xk != 1;
    const bool grads = a.gradient && (a.dw || a.dbias);
    p.kpt = grads ? std::max(1, pow2_ceil(d) / kFewThreads) : 0;
    FewArgs& k = p.k;
    k.x = a.x; k.xr = a.xr; k.xk = a.xk; k.w = a.w; k.wr = a.wr; k.wk = a.wk;
    k.bias = a.bias; k.labels = a.labels; k.n = a.n; k.d = d; k.c = (int)a.c;
    k.weight = a.weight; k.weight_stride = a.weight_stride; k.scale = a.scale;
    k.have_lse = a.have_lse; k.want_dw = a.dw != nullptr;
    k.loss = a.loss; k.lse = a.lse; k.dx = a.dx; k.dxr = a.dxr; k.dxk = a.dxk;
    const int64_t line = p.cols ? a.xk : a.xr;
    const bool unit_inner = p.cols ? a.xr == 1 : a.xk == 1;
    k.vec_ok = unit_inner && (uintptr_t)a.x % 16 == 0 && (line * es) % 16 == 0 && line >= 0;
    k.log_dc = ilog2(std::min(kFewThreads, std::max(32, pow2_ceil(d))));
    p.n_rs = kFewThreads >> k.log_dc;
    // Rows of a tile: what kFewTileBytes hold, at least one vector (a 32-byte sector when the
    // rows are contiguous), and fewer where that would leave SMs without a tile.
    const int least = p.cols ? 32 / es : V;
    int rows = kFewMaxRows;
    while (rows > least && (int64_t)rows * d * es > kFewTileBytes) rows /= 2;
    while (rows > std::max(8, least) && (a.n + rows - 1) / rows < 2 * sms) rows /= 2;
    k.rows = rows; k.log_rows = ilog2(rows);
    // an odd number of 16-byte units between lines: 16-byte reads across lines meet no bank twice
    int units = ((p.cols ? rows : d) + V - 1) / V + 1;
    if (units % 2 == 0) ++units;
    k.pitch = units * V;
    k.n_tiles = (int)((a.n + rows - 1) / rows);
    const size_t tile = ((size_t)(p.cols ? d : rows) * k.pitch * es + 127) / 128 * 128;
    const int slots = rows >= 32 ? kFewThreads / rows : kFewThreads / 32;
    const size_t rest = sizeof(float) * ((size_t)(d + V) * p.cp + (size_t)rows * p.cp * (slots + 1) + p.cp + 16);
    k.stages = 2 * tile + rest <= kFewMaxSmem ? 2 : 1;
    p.smem = k.stages * tile + rest;
    const int per_sm = p.smem <= 112 * 1024 && p.cp * std::max(1, p.kpt) <= 16 ? 2 : 1;
    p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(k.n_tiles, (int64_t)per_sm * sms));
    return p;
}

template <typename T, int CP, int KPT>
cudaError_t few_launch(const FewPlan& p, cudaStream_t stream) {
    auto fn = p.cols ? xent_few_kernel<T, CP, KPT, true> : xent_few_kernel<T, CP, KPT, false>;
    cudaError_t e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem);
    if (e != cudaSuccess) return e;
    KernelTimer kt(stream, GAFIME_KERNEL_XENT);
    fn<<<p.grid, kFewThreads, p.smem, stream>>>(p.k);
    return cudaGetLastError();
}

template <typename T, int CP>
cudaError_t few_launch_k(const FewPlan& p, cudaStream_t s) {
    switch (p.kpt) {
        case 0: return few_launch<T, CP, 0>(p, s);
        case 1: return few_launch<T, CP, 1>(p, s);
        case 2: return few_launch<T, CP, 2>(p, s);
        case 4: return few_launch<T, CP, 4>(p, s);
        case 8:
            if constexpr (CP <= 8) return few_launch<T, CP, 8>(p, s);
    }
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t few_launch_t(const FewPlan& p, const XentCall& a) {
    cudaError_t e = cudaErrorInvalidValue;
    if (a.n > 0) {
        switch (p.cp) {
            case 2: e = few_launch_k<T, 2>(p, a.stream); break;
            case 4: e = few_launch_k<T, 4>(p, a.stream); break;
            case 8: e = few_launch_k<T, 8>(p, a.stream); break;
            case 16: e = few_launch_k<T, 16>(p, a.stream); break;
        }
        if (e != cudaSuccess) return e;
    }
    if (!p.kpt) return cudaSuccess;
    const int64_t size = a.c * a.d;
    const int64_t blocks = (a.dw ? (size + 31) / 32 : 0) + (a.dbias ? (a.c + 31) / 32 : 0);
    KernelTimer kt(a.stream, GAFIME_KERNEL_XENT);
    xent_few_sum_kernel<T><<<(unsigned)blocks, 512, 0, a.stream>>>(
        p.k.part, a.n > 0 ? p.grid * p.n_rs : 0, size, (T*)a.dw, p.k.part_bias, a.n > 0 ? p.grid : 0, (int)a.c, a.dbias);
    return cudaGetLastError();
}

size_t few_carve(const XentCall& a, FewPlan& p, uint8_t* ws) {
    Carver cv(ws);
    if (p.kpt) {
        p.k.part = cv.take<float>(a.dw ? (size_t)p.grid * p.n_rs * a.c * a.d : 0);
        p.k.part_bias = cv.take<float>((size_t)p.grid * a.c);
    }
    return cv.used;
}

}  // namespace

bool xent_few_fits(const XentCall& a) {
    if (a.c > kFewMaxC || a.d > kFewMaxD) return false;
    // running sums of c x (features a thread) in registers, and a tile with w in shared memory
    return std::max(2, pow2_ceil((int)a.c)) * std::max(1, pow2_ceil((int)a.d) / kFewThreads) <= 64 &&
           few_plan(a, 148).smem <= kFewMaxSmem;
}

size_t xent_few_workspace(const XentCall& a, int sms) {
    FewPlan p = few_plan(a, sms);
    return few_carve(a, p, nullptr);
}

cudaError_t xent_few(const XentCall& a, int sms) {
    FewPlan p = few_plan(a, sms);
    few_carve(a, p, a.ws);
    switch (a.type) {
        case GAFIME_TYPE_FP32: return few_launch_t<float>(p, a);
        case GAFIME_TYPE_FP16: return few_launch_t<__half>(p, a);
        default: return few_launch_t<__nv_bfloat16>(p, a);
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

size_t workspace_of(const XentCall& a) {
    const int sms = sm_count_of_current();
    return xent_few_fits(a) ? xent_few_workspace(a, sms) : xent_tc_workspace(a, sms);
}

int run_xent(const XentCall& a) {
    if (gafime_cuda_available() != 1) return GAFIME_ERROR_CUDA_NOT_AVAILABLE;
    if (a.n == 0 && !a.dw && !a.dbias) return GAFIME_SUCCESS;
    const size_t need = workspace_of(a);
    if (need > a.ws_bytes || (need && (!a.ws || (uintptr_t)a.ws % 256))) return GAFIME_ERROR_INVALID_ARGS;
    const int sms = sm_count_of_current();
    const cudaError_t e = xent_few_fits(a) ? xent_few(a, sms) : xent_tc(a, sms);
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
