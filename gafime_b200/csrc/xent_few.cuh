// xent_few.cuh -- softmax cross entropy of a linear head with few classes: one pass over x.
//
// Every logit of a row fits into registers, so loss, dw and dbias (and dx) come from one read of
// x; nothing of size n x c exists.  What bounds it is reading x, as long as its 2 c (loss: c)
// multiply-adds a value and the shared-memory traffic around them keep up: about 5.5 cycles an
// SM for 32 fp32 values at the measured copy rate.
//
// A warp owns a tile of kRowsMost (or fewer) rows x 128 features in shared memory, which it
// fills with its own asynchronous copies; W warps side by side cover the features.  Tiles are
// not double-buffered: a warp that waits for its copies leaves the SM to eleven others, which
// costs no barrier and no second tile.
//   1. a lane is a row: partial dot products with c accumulators, w broadcast from shared memory
//      (fewer rows than lanes: the lanes of a row share the features)
//   2. the W partial logits are added through shared memory (the only barrier); a lane computes
//      its row's softmax, loss and g, and leaves g in shared memory
//   3. a lane is four features: c x 4 sums of g x over the tile's rows
// Without gradients a warp walks over the features by itself, and there is no barrier at all.
// The sums of step 3 move to a partial in global memory every kFlushRows rows: short fp32
// chains, added in fp64 in a fixed order by xent_few_sum_kernel at the end.
//
// Tile layout: 16-byte units, unit q of line L at q ^ (L >> shift & mask), so that both the
// reads along lines and those across them meet no bank twice.  A line is a row (x row by row)
// or a feature (x column by column, as buckets hold it).
#pragma once

#include <math.h>

#include "engine.h"
#include "xent.h"

namespace gafime {

constexpr int kFewFeatures = 128;     // of a warp's tile
constexpr int kRowsMost = 32;
constexpr int kFlushRows = 256;

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
    int have_lse;
    float* loss;
    float* lse;
    void* dx;
    int64_t dxr, dxk;
    float* part;         // [groups][c][d_pad]
    double* part_bias;   // [groups][c]
    int d_pad;           // features rounded up to whole tiles
    int rows, log_rows;  // of a tile: 8, 16 or 32
    int vec_ok;          // 16-byte copies allowed
    int warps;           // W, side by side
    int groups;          // of W warps in a CTA
    int n_tiles;         // of rows
};

struct FewPlan {
    FewArgs k;
    int cp, grid, threads;
    bool cols, grad;
    size_t smem;
};

// One per type (xent_few_*.cu): launches the kernel of the plan.
cudaError_t few_launch_fp32(const FewPlan& p, cudaStream_t s);
cudaError_t few_launch_fp16(const FewPlan& p, cudaStream_t s);
cudaError_t few_launch_bf16(const FewPlan& p, cudaStream_t s);

namespace few {

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Geometry of a tile: bytes of a line, and the exchange of its 16-byte units.
template <typename T, bool COLS>
struct Tile {
    int line_bytes, shift, mask;
    __device__ explicit Tile(int rows) {
        line_bytes = (COLS ? rows : kFewFeatures) * (int)sizeof(T);
        const int units = line_bytes / 16;                    // of a line
        mask = units >= 8 ? 7 : units - 1;
        shift = units >= 8 ? 0 : units == 4 ? 1 : units == 2 ? 2 : 3;
    }
    // byte offset of element e of line l
    __device__ __forceinline__ int at(int l, int e) const {
        const int b = e * (int)sizeof(T);
        return l * line_bytes + (((b >> 4) ^ ((l >> shift) & mask)) << 4) + (b & 15);
    }
};

// Queue a warp's copies of rows [r0, r0 + R) x features [k0, k0 + 128).  Rows and features past
// the table read zero in units that hold some of it; other units are never used.
template <typename T, bool COLS>
__device__ __forceinline__ void load_tile(const FewArgs& a, const Tile<T, COLS>& g, uint8_t* tile, int64_t r0, int k0,
                                          int lane) {
    constexpr int V = 16 / sizeof(T);
    const int left = (int)min((int64_t)a.rows, a.n - r0), feats = min(kFewFeatures, a.d - k0);
    const T* x = (const T*)a.x + r0 * a.xr + (int64_t)k0 * a.xk;
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(tile);
    const int lines = COLS ? feats : left, len = COLS ? left : feats;
    const int64_t ls = COLS ? a.xk : a.xr, es = COLS ? a.xr : a.xk;
    if (a.vec_ok) {
        const int units = COLS ? a.rows / V : (feats + V - 1) / V;
        if (COLS || units == kFewFeatures / V) {
            // a power of two of units to a line
            const int lu = COLS ? a.log_rows - (sizeof(T) == 4 ? 2 : 3) : (sizeof(T) == 4 ? 5 : 4);
            for (int i = lane; i < (lines << lu); i += 32) {
                const int l = i >> lu, q = i & ((1 << lu) - 1);
                const int bytes = max(0, min(V, len - q * V)) * (int)sizeof(T);
                copy16(dst + g.at(l, q * V), bytes ? x + l * ls + q * V : x, bytes);
            }
        } else {
            for (int l = 0; l < lines; ++l)
                for (int q = lane; q < units; q += 32) {
                    const int bytes = min(V, len - q * V) * (int)sizeof(T);
                    copy16(dst + g.at(l, q * V), x + l * ls + q * V, bytes);
                }
        }
    } else {
        // any strides: element by element, neighbouring lanes on neighbouring elements
        const int full = COLS ? a.rows : (feats + V - 1) / V * V;
        for (int l = 0; l < lines; ++l)
            for (int e = lane; e < full; e += 32) {
                if constexpr (sizeof(T) == 4) {
                    copy4(dst + g.at(l, e), e < len ? x + l * ls + e * es : x, e < len ? 4 : 0);
                } else {
                    *reinterpret_cast<T*>(tile + g.at(l, e)) = e < len ? x[l * ls + e * es] : from_float<T>(0.f);
                }
            }
    }
    if (!COLS && left < a.rows) {
        // rows past the table: their lanes read them in step 1
        for (int l = left; l < a.rows; ++l)
            for (int q = lane; q < kFewFeatures / V; q += 32)
                *reinterpret_cast<uint4*>(tile + g.at(l, q * V)) = make_uint4(0, 0, 0, 0);
    }
}

// CP floats, of which the first C count, from a line of whole float4 (float2 for two)
template <int C>
struct Line {
    static constexpr int kPitch = C <= 2 ? 2 : (C + 3) / 4 * 4;
};
template <int C>
__device__ __forceinline__ void load_line(float (&v)[C], const float* p) {
    if constexpr (C == 2) {
        const float2 t = *reinterpret_cast<const float2*>(p);
        v[0] = t.x;
        v[1] = t.y;
    } else {
        #pragma unroll
        for (int c = 0; c < C; c += 4) {
            const float4 t = *reinterpret_cast<const float4*>(p + c);
            v[c] = t.x;
            if (c + 1 < C) v[c + 1] = t.y;
            if (c + 2 < C) v[c + 2] = t.z;
            if (c + 3 < C) v[c + 3] = t.w;
        }
    }
}

// 4 neighbouring elements (8-byte units in 16 bits)
__device__ __forceinline__ void load4(float (&v)[4], const uint8_t* p, float) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x;
    v[1] = t.y;
    v[2] = t.z;
    v[3] = t.w;
}
__device__ __forceinline__ void load4(float (&v)[4], const uint8_t* p, __half) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&t.x));
    const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
    v[0] = f.x;
    v[1] = f.y;
    v[2] = g.x;
    v[3] = g.y;
}
__device__ __forceinline__ void load4(float (&v)[4], const uint8_t* p, __nv_bfloat16) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(t.x << 16);
    v[1] = __uint_as_float(t.x & 0xffff0000u);
    v[2] = __uint_as_float(t.y << 16);
    v[3] = __uint_as_float(t.y & 0xffff0000u);
}

// C: classes the code has room for (a.c of them exist); GRAD: dw and dbias wanted or dx
template <typename T, int C, bool COLS, bool GRAD, bool DX>
__global__ void __launch_bounds__(512, 1) xent_few_kernel(const FewArgs a) {
    constexpr int CL = Line<C>::kPitch;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int W = a.warps, group = warp / W, wg = warp - group * W;   // warp wg of its group
    const int R = a.rows;
    const Tile<T, COLS> geo(R);
    const int warps = W * a.groups;
    const int tile_bytes = R * kFewFeatures * (int)sizeof(T);
    uint8_t* tile = smem + (size_t)warp * tile_bytes;
    float* ws = reinterpret_cast<float*>(smem + (size_t)warps * tile_bytes);   // w: [d_pad][CL]
    float* gs = ws + (size_t)a.d_pad * CL + (size_t)warp * (GRAD ? kRowsMost * CL : 0);   // g: [rows][CL], a warp's own
    float* red = ws + (size_t)a.d_pad * CL + (size_t)warps * (GRAD ? kRowsMost * CL : 0);   // [2][groups][W][C][32]
    double* bsum = reinterpret_cast<double*>(red + (W > 1 ? 2 * (size_t)warps * C * 32 : 0)) +
                   (size_t)group * C * 32;                                                  // bias: [C][32] a group

    for (int i = threadIdx.x; i < a.d_pad * CL; i += blockDim.x) {
        const int k = i / CL, c = i % CL;
        ws[i] = c < a.c && k < a.d ? to_float(((const T*)a.w)[c * a.wr + k * a.wk]) : 0.f;
    }
    float bias[C];
    #pragma unroll
    for (int c = 0; c < C; ++c) bias[c] = c < a.c ? (a.bias ? a.bias[c] : 0.f) : -INFINITY;
    if (GRAD && wg == 0)
        for (int c = 0; c < C; ++c) bsum[c * 32 + lane] = 0.0;
    __syncthreads();

    float acc[GRAD ? 4 : 1][C], db[C];
    #pragma unroll
    for (int f = 0; f < (GRAD ? 4 : 1); ++f)
        #pragma unroll
        for (int c = 0; c < C; ++c) acc[f][c] = 0.f;
    #pragma unroll
    for (int c = 0; c < C; ++c) db[c] = 0.f;

    const int row = lane & (R - 1), share = lane >> a.log_rows, shares = 32 >> a.log_rows;
    const int kw = wg * kFewFeatures;                      // GRAD: the warp's features
    // the groups of all CTAs take tiles in turn, one group of every CTA first
    const int64_t first = (int64_t)group * gridDim.x + blockIdx.x, step = (int64_t)a.groups * gridDim.x;
    const size_t part_at = (size_t)first * a.c * a.d_pad;
    int parity = 0, since = 0;
    bool flushed = false;

    // sums so far to the group's partial
    auto flush = [&]() {
        if (a.part) {
            #pragma unroll
            for (int f = 0; f < (GRAD ? 4 : 1); ++f) {
                const int k = kw + (COLS ? lane + 32 * f : 4 * lane + f);
                #pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (c < a.c) {
                        float* p = a.part + part_at + (size_t)c * a.d_pad + k;
                        *p = flushed ? *p + acc[f][c] : acc[f][c];
                    }
                    acc[f][c] = 0.f;
                }
            }
        }
        if (wg == 0)
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                bsum[c * 32 + lane] += (double)db[c];
                db[c] = 0.f;
            }
        flushed = true;
        since = 0;
    };

    for (int64_t t = first; t < a.n_tiles; t += step) {
        const int64_t r0 = t * R, gr = r0 + row;
        float z[C];
        #pragma unroll
        for (int c = 0; c < C; ++c) z[c] = 0.f;
        int64_t y64 = -1;
        float rw = 0.f, shift_in = 0.f;
        for (int k0 = GRAD ? kw : 0; k0 < a.d; k0 += GRAD ? a.d_pad : kFewFeatures) {
            __syncwarp();                                  // the tile's last readers are done
            load_tile<T, COLS>(a, geo, tile, r0, k0, lane);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (k0 == (GRAD ? kw : 0) && gr < a.n) {       // meanwhile
                y64 = a.labels[gr];
                if (GRAD) rw = (a.weight ? a.weight[gr * a.weight_stride] : 1.f) * a.scale;
                if (a.have_lse) shift_in = a.lse[gr];
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            // 1. a lane is a row
            const int feats = min(kFewFeatures, a.d - k0);
            const float* wk = ws + (size_t)k0 * CL;
            if (COLS) {
                #pragma unroll 4
                for (int k = share; k < feats; k += shares) {
                    const float xv = to_float(*reinterpret_cast<const T*>(tile + geo.at(k, row)));
                    float wv[C];
                    load_line<C>(wv, wk + k * CL);
                    #pragma unroll
                    for (int c = 0; c < C; ++c) z[c] = fmaf(xv, wv[c], z[c]);
                }
            } else {
                #pragma unroll 2
                for (int k = share * 4; k < feats; k += shares * 4) {
                    float xv[4];
                    load4(xv, tile + geo.at(row, k), T{});
                    #pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        float wv[C];
                        load_line<C>(wv, wk + (k + v) * CL);
                        #pragma unroll
                        for (int c = 0; c < C; ++c) z[c] = fmaf(xv[v], wv[c], z[c]);
                    }
                }
            }
        }
        for (int o = R; o < 32; o <<= 1)
            #pragma unroll
            for (int c = 0; c < C; ++c) z[c] += __shfl_xor_sync(0xffffffffu, z[c], o);
        // 2. logits of all warps, softmax, loss, g
        if (GRAD && W > 1) {
            float* mine = red + ((size_t)(parity * a.groups + group) * W) * C * 32;
            #pragma unroll
            for (int c = 0; c < C; ++c) mine[(wg * C + c) * 32 + lane] = z[c];
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(W * 32) : "memory");
            #pragma unroll
            for (int c = 0; c < C; ++c) z[c] = 0.f;
            for (int w = 0; w < W; ++w)
                #pragma unroll
                for (int c = 0; c < C; ++c) z[c] += mine[(w * C + c) * 32 + lane];
            parity ^= 1;
        }
        const bool kept = y64 >= 0;
        const int y = kept && y64 < a.c ? (int)y64 : -1;   // kept with y < 0: no such class
        float m = -INFINITY, zy = NAN, s = 0.f;
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            z[c] += bias[c];
            m = fmaxf(m, z[c]);
            if (c == y) zy = z[c];
        }
        if (m == -INFINITY) m = 0.f;                       // every class excluded: exp(-inf) = 0, not NaN
        float e[C];
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            e[c] = expf(z[c] - m);
            s += e[c];
        }
        const float ls = logf(s);
        if (wg == 0 && share == 0 && gr < a.n && !a.have_lse) {
            a.loss[gr] = kept ? (m - zy) + ls : 0.f;
            if (a.lse) a.lse[gr] = kept ? m + ls : 0.f;
        }
        if (GRAD) {
            // with this call's own sum, e / s; else exp of the difference to the given lse
            const float inv = 1.f / s;
            const uint32_t mask = __ballot_sync(0xffffffffu, kept);   // bit r (r + R, ...): row r counts
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                const float p = a.have_lse ? expf(z[c] - shift_in) : e[c] * inv;
                float g = kept ? (p - (c == y ? 1.f : 0.f)) * rw : 0.f;
                if (kept && y < 0) g = NAN;
                if (c >= a.c) g = 0.f;
                e[c] = g;
                if (share == 0) {
                    gs[row * CL + c] = g;
                    db[c] += g;
                }
            }
            __syncwarp();
            if (DX) {
                const int left = (int)min((int64_t)R, a.n - r0), feats = min(kFewFeatures, a.d - kw);
                T* dx = (T*)a.dx + r0 * a.dxr + (int64_t)kw * a.dxk;
                const float* wk = ws + (size_t)kw * CL;
                if (COLS) {
                    // neighbouring lanes are neighbouring rows
                    if (row < left)
                        for (int k = share; k < feats; k += shares) {
                            float wv[C], v = 0.f;
                            load_line<C>(wv, wk + k * CL);
                            #pragma unroll
                            for (int c = 0; c < C; ++c) v = fmaf(e[c], wv[c], v);
                            dx[row * a.dxr + k * a.dxk] = from_float<T>(kept ? v : 0.f);
                        }
                } else {
                    for (int k = lane; k < feats; k += 32) {
                        float wv[C];
                        load_line<C>(wv, wk + k * CL);
                        #pragma unroll 4
                        for (int r = 0; r < left; ++r) {
                            float g[C], v = 0.f;
                            load_line<C>(g, gs + r * CL);
                            #pragma unroll
                            for (int c = 0; c < C; ++c) v = fmaf(g[c], wv[c], v);
                            dx[r * a.dxr + k * a.dxk] = from_float<T>((mask >> r) & 1 ? v : 0.f);
                        }
                    }
                }
            }
            // 3. a lane is four features
            if (a.part && mask) {
                const uint32_t all = R == 32 ? 0xffffffffu : (1u << R) - 1;
                if (COLS) {
                    const int feats = min(kFewFeatures, a.d - kw);
                    auto sums = [&](bool whole) {
                        #pragma unroll 2
                        for (int r = 0; r < R; r += 4) {
                            #pragma unroll
                            for (int f = 0; f < 4; ++f) {
                                if (32 * f >= feats) break;
                                float xv[4];
                                load4(xv, tile + geo.at(lane + 32 * f, r), T{});
                                #pragma unroll
                                for (int v = 0; v < 4; ++v) {
                                    // what a left-out row holds may be no number
                                    const float xk = whole || ((mask >> (r + v)) & 1) ? xv[v] : 0.f;
                                    float g[C];
                                    load_line<C>(g, gs + (r + v) * CL);
                                    #pragma unroll
                                    for (int c = 0; c < C; ++c) acc[f][c] = fmaf(g[c], xk, acc[f][c]);
                                }
                            }
                        }
                    };
                    if ((mask & all) == all)
                        sums(true);
                    else
                        sums(false);
                } else {
                    #pragma unroll 4
                    for (int r = 0; r < R; ++r) {
                        if (!((mask >> r) & 1)) continue;
                        float xv[4], g[C];
                        load4(xv, tile + geo.at(r, 4 * lane), T{});
                        load_line<C>(g, gs + r * CL);
                        #pragma unroll
                        for (int f = 0; f < 4; ++f)
                            #pragma unroll
                            for (int c = 0; c < C; ++c) acc[f][c] = fmaf(g[c], xv[f], acc[f][c]);
                    }
                }
            }
            since += R;
            if (since >= kFlushRows) flush();
        }
    }
    if (GRAD) {
        if (since > 0 || !flushed) flush();
        if (wg == 0)
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                double v = bsum[c * 32 + lane];
                #pragma unroll
                for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
                if (lane == 0 && c < a.c) a.part_bias[(size_t)first * a.c + c] = v;
            }
    }
}

template <typename T, int C, bool COLS, bool GRAD, bool DX>
cudaError_t launch(const FewPlan& p, cudaStream_t stream) {
    auto fn = xent_few_kernel<T, C, COLS, GRAD, DX>;
    const cudaError_t e =
        cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem);
    if (e != cudaSuccess) return e;
    KernelTimer kt(stream, GAFIME_KERNEL_XENT);
    fn<<<p.grid, p.threads, p.smem, stream>>>(p.k);
    return cudaGetLastError();
}

template <typename T, int C>
cudaError_t launch_c(const FewPlan& p, cudaStream_t s) {
    if (!p.grad) return p.cols ? launch<T, C, true, false, false>(p, s) : launch<T, C, false, false, false>(p, s);
    if (!p.k.dx) return p.cols ? launch<T, C, true, true, false>(p, s) : launch<T, C, false, true, false>(p, s);
    return p.cols ? launch<T, C, true, true, true>(p, s) : launch<T, C, false, true, true>(p, s);
}

template <typename T>
cudaError_t launch_t(const FewPlan& p, cudaStream_t s) {
    switch (p.cp) {
        case 2: return launch_c<T, 2>(p, s);
        case 3: return launch_c<T, 3>(p, s);
        case 4: return launch_c<T, 4>(p, s);
        case 6: return launch_c<T, 6>(p, s);
        case 8: return launch_c<T, 8>(p, s);
        case 16: return launch_c<T, 16>(p, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace few

}  // namespace gafime
