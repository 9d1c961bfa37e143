// xent_few.cuh -- softmax cross entropy of a linear head with few classes: one pass over x.
//
// Every logit of a row fits into registers, so loss, dw and dbias (and dx) come from one read of
// x; nothing of size n x c exists.  What bounds it is reading x, as long as its 2 c (loss: c)
// multiply-adds a value and the shared-memory traffic around them keep up: about 5.5 cycles an
// SM for 32 fp32 values at the measured copy rate.
//
// A warp owns a tile of 32 rows (fewer in small calls) x 64 or 128 features in shared memory,
// which it fills with its own asynchronous copies; W warps side by side cover the features.
// Tiles are not double-buffered: a warp that waits for its copies leaves the SM to up to 23
// others, which costs no second tile (measured against two buffers of half the
// rows: 64-byte pieces of columns instead of 128 cost more than the overlap gained).
//   1. a lane is a row: partial dot products with c accumulators, w broadcast from shared memory
//      (fewer rows than lanes: the lanes of a row share the features)
//   2. the W partial logits are added through shared memory (the only barrier); a lane computes
//      its row's softmax, loss and g, and leaves g in shared memory
//   3. a lane is two or four features: c sums each of g x over the tile's rows (a whole tile, past
//      the table's features too: those sums are not read)
// Without gradients a warp walks over the features by itself, without that barrier.
// The sums of step 3 move to a partial in global memory every kFlushRows rows: short fp32
// chains, added in fp64 in a fixed order by xent_few_sum_kernel at the end.
//
// Measured on a B200 (copy rate 6,551 GB/s): steps of 1e6 x 256 with 2 classes 0.176 ms by rows
// (5,900 GB/s) and 0.182 ms by columns (5,700), of 4e6 x 128 with 3 classes 0.37 and 0.36 ms; their
// losses 0.168 and 0.163 (6,350), 0.33 and 0.31 ms (6,650); the loss of 300001 x 2048 with 5 classes
// 0.40 ms by rows.  Narrow tables are bound by a row's own work (softmax, g, the sums of lanes): the
// step of 4e6 x 16 with 2 classes 0.139 ms.  From six classes on the multiply-adds bound it:
// 500000 x 512 with 8 classes takes 0.45 ms by rows, 0.52 by columns.
//
// Tile layout: 16-byte units, unit q of line L at q ^ (L >> shift & mask), so that both the
// reads along lines and those across them meet no bank twice.  A line is a row (x row by row)
// or a feature (x column by column, as buckets hold it).
#pragma once

#include <math.h>

#include "engine.h"
#include "xent.h"

namespace gafime {

// Most classes of this path.  With gradients 8: at 16 their sums leave no registers (200000 x 1024
// fp32: 1.5 to 3.1 ms a step, the tensor cores' path 1.16 ms); without, 16 (0.31 ms against 0.72).
constexpr int kFewMaxC = 16, kFewMaxGrad = 8;
// Features of a warp's tile: 128 with gradients, 64 without and for narrow tables (up to 24 warps
// an SM in place of 12 to 16: steps of 4e6 x 16 with 2 classes 217 -> 174 us, 500000 x 33 with 8
// classes 102 -> 67).
constexpr int few_features(bool grad, bool narrow) { return grad && !narrow ? 128 : 64; }
// Warps that an SM holds, by registers: 24 of 80, 20 of 96 or 16 of 128.
constexpr int few_warps(int c, int features, bool grad) {
    return features == 128 || c >= 6 ? 16 : grad && c > 2 ? 20 : 24;
}
// Threads of a CTA, at most.
constexpr int few_threads(int features, bool grad) { return features == 128 ? 512 : grad ? 128 : 256; }
constexpr int kRowsMost = 32;
// Losses by columns: tiles side by side for 4 classes and 32 features or more (below; with more
// classes or fewer features the barriers cost more: 500000 x 512 with 8 classes 187 -> 200 us,
// 4e6 x 16 with 2 classes 72 -> 78).
constexpr int kBesideMaxC = 4, kBesideMinD = 32;
constexpr int kFlushRows = 256;
constexpr size_t kFewMaxSmem = 226 * 1024;   // of a CTA, at most

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
    int have_lse;        // loss and lse are there already
    float* loss;
    float* lse;
    void* dx;
    int64_t dxr, dxk;
    float* part;         // [groups][c][d_pad]
    double* part_bias;   // [groups][c]
    int d_pad;           // features rounded up to whole tiles
    int rows, log_rows;  // of a tile: 8, 16 or 32
    int warps;           // W, side by side
    int groups;          // of W warps in a CTA
    int n_tiles;         // of rows
};

struct FewPlan {
    FewArgs k;
    int cp, grid, threads, features;
    bool cols, grad;
    int beside;          // groups whose tiles lie side by side (by columns, with gradients), or 1
    bool vec;            // 16-byte copies of x: unit stride, aligned lines
    size_t smem;
};

// Launches the kernel of the plan: one per type (the last argument names it) and order of x, each
// in a file of its own (xent_few_*.cu), which compile side by side.
cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, float);
cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, __half);
cudaError_t few_launch_rows(const FewPlan& p, cudaStream_t s, __nv_bfloat16);
cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, float);
cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, __half);
cudaError_t few_launch_columns(const FewPlan& p, cudaStream_t s, __nv_bfloat16);

namespace few {

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Geometry of a tile of R rows (of G groups' tiles side by side, by columns): bytes of a line, and
// the exchange of its 16-byte units.  The pattern repeats every 8 lines, so unrolled loops need a
// few precomputed offsets only.
template <typename T, bool COLS, int R, int F, int G = 1>
struct Tile {
    static constexpr int kLine = (COLS ? G * R : F) * (int)sizeof(T);
    static constexpr int kUnits = kLine / 16;                 // of a line
    static constexpr int kMask = kUnits >= 8 ? 7 : kUnits - 1;
    static constexpr int kShift = kUnits >= 8 ? 0 : kUnits == 4 ? 1 : kUnits == 2 ? 2 : 3;
    // byte offset of unit q of line l
    static __device__ __forceinline__ int unit(int l, int q) { return l * kLine + ((q ^ ((l >> kShift) & kMask)) << 4); }
    // byte offset of element e of line l
    static __device__ __forceinline__ int at(int l, int e) {
        const int b = e * (int)sizeof(T);
        return unit(l, b >> 4) + (b & 15);
    }
};

// The same for any strides: element by element, neighbouring lanes on neighbouring elements of a
// line (or of several short lines), eight loads under way.
template <typename T, bool COLS, int R, int F>
__device__ __forceinline__ void load_tile_any(const FewArgs& a, uint8_t* tile, int64_t r0, int k0, int lane) {
    using Geo = Tile<T, COLS, R, F>;
    constexpr int V = 16 / sizeof(T);
    const int left = (int)min((int64_t)R, a.n - r0), feats = min(F, a.d - k0);
    const T* x = (const T*)a.x + r0 * a.xr + (int64_t)k0 * a.xk;
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(tile);
    const int lines = COLS ? feats : left, len = COLS ? left : feats;
    const int64_t ls = COLS ? a.xk : a.xr, es = COLS ? a.xr : a.xk;
    constexpr int E = COLS ? R : F, W = E < 32 ? E : 32;  // elements of a line, and of those at a time
    constexpr int L = 32 / W;                             // lines at a time
    const int full = COLS ? R : (feats + V - 1) / V * V;
    const int e0 = lane % W, l0 = lane / W;
    for (int h = 0; h < E / W; ++h) {
        const int e = e0 + h * W;
        if (e >= full) break;
        const bool in = e < len;
        const T* src = x + l0 * ls + (in ? e * es : 0);
        const int64_t hop = L * ls;
        const int unit = e * (int)sizeof(T) >> 4, rest = e * (int)sizeof(T) & 15;
        if constexpr (sizeof(T) == 4) {
            #pragma unroll 8
            for (int l = l0; l < lines; l += L, src += hop) copy4(dst + Geo::unit(l, unit) + rest, in ? src : x, in ? 4 : 0);
        } else {
            for (int l = l0; l < lines; l += 8 * L) {
                T v[8];
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = from_float<T>(0.f);
                    if (in && l + i * L < lines) v[i] = src[i * hop];
                }
                src += 8 * hop;
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (l + i * L < lines) *reinterpret_cast<T*>(tile + Geo::unit(l + i * L, unit) + rest) = v[i];
            }
        }
    }
}

// Queue a warp's copies of rows [r0, r0 + R) x features [k0, k0 + 128).  Rows and features past
// the table read zero in units that hold some of it; other units are never used.
template <typename T, bool COLS, int R, int F, bool VEC>
__device__ __forceinline__ void load_tile(const FewArgs& a, uint8_t* tile, int64_t r0, int k0, int lane) {
    using Geo = Tile<T, COLS, R, F>;
    constexpr int V = 16 / sizeof(T), U = Geo::kUnits;
    constexpr int LS = U >= 32 ? 1 : 32 / U;                  // lines a warp covers at a time
    const int left = (int)min((int64_t)R, a.n - r0), feats = min(F, a.d - k0);
    const T* x = (const T*)a.x + r0 * a.xr + (int64_t)k0 * a.xk;
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(tile);
    const int lines = COLS ? feats : left, len = COLS ? left : feats;
    const int64_t ls = COLS ? a.xk : a.xr;
    if constexpr (VEC) {
        const int l0 = lane / U, q = lane % U;
        const int bytes = max(0, min(V, len - q * V)) * (int)sizeof(T);
        const T* src = x + l0 * ls + (bytes ? q * V : 0);
        const int64_t hop = LS * ls;
        if (bytes || COLS) {
            // l0 and j LS share no bit, so the exchange splits into a lane's part and j's
            const int own = l0 * Geo::kLine + ((q ^ ((l0 >> Geo::kShift) & Geo::kMask)) << 4);
            constexpr int kAll = (COLS ? F : R) / LS;
            if (lines == (COLS ? F : R)) {
                #pragma unroll 8
                for (int j = 0; j < kAll; ++j, src += hop)
                    copy16(dst + j * LS * Geo::kLine + (own ^ ((((j * LS) >> Geo::kShift) & Geo::kMask) << 4)), src, bytes);
            } else {
                for (int j = 0; l0 + j * LS < lines; ++j, src += hop)
                    copy16(dst + j * LS * Geo::kLine + (own ^ ((((j * LS) >> Geo::kShift) & Geo::kMask) << 4)), src, bytes);
            }
        }
    } else {
        load_tile_any<T, COLS, R, F>(a, tile, r0, k0, lane);
    }
    if (!COLS && left < R) {
        // rows past the table: their lanes read them in step 1
        for (int l = left; l < R; ++l)
            for (int q = lane; q < U; q += 32) *reinterpret_cast<uint4*>(tile + Geo::unit(l, q)) = make_uint4(0, 0, 0, 0);
    }
}

// The tiles of G groups side by side, x by columns: the groups' warps over the same features fill
// one tile of G x 32 rows together.  A column is then read in pieces of 512 bytes (fp32, four
// groups) in place of 128; by columns that lie pages apart it costs less than the two barriers
// of the CTA that it takes.  Steps by columns, fp32, apart and side by side: 4e6 x 128 with 3
// classes 502 and 411 us, 1e6 x 256 with 2 classes 226 and 195; 2e6 x 50 151 and 156; losses 441
// and 314, 190 and 163, 78 and 72.
template <typename T, int F, int G>
__device__ __forceinline__ void load_side_by_side(const FewArgs& a, uint8_t* tile, int64_t r0, int k0, int group, int lane) {
    using Geo = Tile<T, true, 32, F, G>;
    constexpr int V = 16 / sizeof(T), U = Geo::kUnits, LS = 32 / U;   // LS: lines of a warp at a time
    const int len = (int)min((int64_t)(32 * G), a.n - r0), feats = min(F, a.d - k0);
    const int l0 = lane / U, q = lane % U;
    const int bytes = max(0, min(V, len - q * V)) * (int)sizeof(T);
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(tile);
    const T* src = (const T*)a.x + r0 * a.xr + (int64_t)(k0 + group * LS + l0) * a.xk + (bytes ? q * V : 0);
    const int64_t hop = (int64_t)LS * G * a.xk;
    #pragma unroll 8
    for (int l = group * LS + l0; l < feats; l += LS * G, src += hop)
        copy16(dst + Geo::unit(l, q), bytes ? src : (const T*)a.x, bytes);
}

// Classes of a line in shared memory, padded so that C pairs are whole 16-byte units.
template <int C>
constexpr int padded() { return (C + 1) / 2 * 2; }
// C pairs from 16-byte units
template <int C>
__device__ __forceinline__ void load_pairs(Pair (&v)[C], const float* p) {
    const ulonglong2* q = reinterpret_cast<const ulonglong2*>(p);
    #pragma unroll
    for (int c = 0; c < C; c += 2) {
        const ulonglong2 t = q[c / 2];
        v[c] = t.x;
        if (c + 1 < C) v[c + 1] = t.y;
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

__device__ __forceinline__ void load_some(float (&v)[2], const uint8_t* p, float) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x;
    v[1] = t.y;
}
__device__ __forceinline__ void load_some(float (&v)[2], const uint8_t* p, __half) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(p));
    v[0] = t.x;
    v[1] = t.y;
}
__device__ __forceinline__ void load_some(float (&v)[2], const uint8_t* p, __nv_bfloat16) {
    const uint32_t t = *reinterpret_cast<const uint32_t*>(p);
    v[0] = __uint_as_float(t << 16);
    v[1] = __uint_as_float(t & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ void load_some(float (&v)[4], const uint8_t* p, T t) {
    load4(v, p, t);
}

// The row of its tile that a lane finishes in step 2 (lanes past R share one).
//   columns: lane = share G + group; it multiplies rows 4 group .. 4 group + 3 (16 bytes of a
//            line) and keeps the one that its share names
//   rows:    lane = share R + row; it multiplies that row alone (four rows a lane, the columns'
//            way, measured the same at 2 classes and slower from 6 on)
template <bool COLS, int R>
struct Lanes {
    static constexpr int kGroups = R / 4, kShares = COLS ? 32 / kGroups : 32 / R;
    static __device__ __forceinline__ int row(int lane) {
        return COLS ? 4 * (lane % kGroups) + ((lane / kGroups) & 3) : lane % R;
    }
};

// Step 1: dot products of the tile's rows with w, all of row Lanes::row(lane) in z at the end.
// w: columns [features][classes], pairs of rows multiplied together, a value of w for four rows;
// rows [feature pairs][classes][2], pairs of features.
template <typename T, int C, bool COLS, int R, int F, int G = 1>
__device__ __forceinline__ void dots(float (&z)[C], const uint8_t* tile, const float* w, int feats, int lane, int beside = 0) {
    using Geo = Tile<T, COLS, R, F, G>;
    using L = Lanes<COLS, R>;
    constexpr int CL = padded<C>(), S = L::kShares;
    if constexpr (COLS) {
        constexpr int K = L::kGroups, B = C <= 6 ? C : 4;     // B: classes at a time
        const int group = lane % K, share = lane / K, own = beside * R + 4 * group;
        #pragma unroll
        for (int c0 = 0; c0 < C; c0 += B) {
            float part[4][B];
            constexpr int Q = C <= 4 ? 2 : 1;   // sets of sums, of alternate lines: shorter chains
            Pair sum[Q][2][B];
            #pragma unroll
            for (int q = 0; q < Q; ++q)
                #pragma unroll
                for (int c = 0; c < B; ++c) sum[q][0][c] = sum[q][1][c] = 0;
            // lines share, share + S, ...: S a multiple of 4, so two exchanges in turn
            const uint8_t* p0 = tile + Geo::at(share, own);
            const uint8_t* p1 = tile + Geo::at(share + S, own);
            const float* wk = w + share * CL + c0;
            auto line = [&](const uint8_t* p, const float* wl, Pair (&to)[2][B]) {
                float xv[4], wv[B];
                load4(xv, p, T{});
                #pragma unroll
                for (int c = 0; c < B; c += 2) {
                    const float2 t = *reinterpret_cast<const float2*>(wl + c);
                    wv[c] = t.x;
                    if (c + 1 < B) wv[c + 1] = t.y;
                }
                const Pair a = pair(xv[0], xv[1]), b = pair(xv[2], xv[3]);
                #pragma unroll
                for (int c = 0; c < B; ++c) {
                    const Pair ww = pair(wv[c], wv[c]);
                    to[0][c] = fma2(a, ww, to[0][c]);
                    to[1][c] = fma2(b, ww, to[1][c]);
                }
            };
            int k = share;
            #pragma unroll 4
            for (; k + S < feats; k += 2 * S) {
                line(p0, wk, sum[0]);
                line(p1, wk + S * CL, sum[Q - 1]);
                p0 += 2 * S * Geo::kLine;
                p1 += 2 * S * Geo::kLine;
                wk += 2 * S * CL;
            }
            if (k < feats) line(p0, wk, sum[0]);
            if constexpr (Q == 2) {
                #pragma unroll
                for (int h = 0; h < 2; ++h)
                    #pragma unroll
                    for (int c = 0; c < B; ++c) {
                        float l0, h0, l1, h1;
                        unpair(l0, h0, sum[0][h][c]);
                        unpair(l1, h1, sum[1][h][c]);
                        sum[0][h][c] = pair(l0 + l1, h0 + h1);
                    }
            }
            #pragma unroll
            for (int c = 0; c < B; ++c) {
                unpair(part[0][c], part[1][c], sum[0][0][c]);
                unpair(part[2][c], part[3][c], sum[0][1][c]);
            }
            // the lane keeps row i = share & 3 of its four: the first two steps of the sum over the
            // lanes halve what is held, as in column_sums
            #pragma unroll
            for (int c = 0; c < B; ++c) {
                const bool odd = share & 1, high = share & 2;
                const float s0 = odd ? part[0][c] : part[1][c], k0 = odd ? part[1][c] : part[0][c];
                const float s1 = odd ? part[2][c] : part[3][c], k1 = odd ? part[3][c] : part[2][c];
                const float u0 = k0 + __shfl_xor_sync(0xffffffffu, s0, K), u1 = k1 + __shfl_xor_sync(0xffffffffu, s1, K);
                float t = (high ? u1 : u0) + __shfl_xor_sync(0xffffffffu, high ? u0 : u1, 2 * K);
                #pragma unroll
                for (int o = 4 * K; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
                if (c0 + c < C) z[c0 + c] += t;
            }
        }
    } else {
        constexpr int V = 16 / sizeof(T);
        const int row = lane % R, share = lane / R, x0 = row & 7;
        const uint8_t* line = tile + row * Geo::kLine;
        Pair sum[C], wv[C];
        #pragma unroll
        for (int c = 0; c < C; ++c) sum[c] = 0;
        // a unit of V features; w is zero past the features, and so is x up to a whole unit
        #pragma unroll 4
        for (int q = share; q * V < feats; q += S) {
            #pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                float xv[4];
                load4(xv, line + ((q ^ x0) << 4) + 8 * h, T{});
                #pragma unroll
                for (int v = 0; v < 4; v += 2) {
                    const Pair x = pair(xv[v], xv[v + 1]);
                    load_pairs<C>(wv, w + (q * V + 4 * h + v) * CL);
                    #pragma unroll
                    for (int c = 0; c < C; ++c) sum[c] = fma2(x, wv[c], sum[c]);
                }
            }
        }
        #pragma unroll
        for (int c = 0; c < C; ++c) {
            float lo, hi;
            unpair(lo, hi, sum[c]);
            float t = lo + hi;
            #pragma unroll
            for (int o = R; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            z[c] += t;
        }
    }
}

// Step 3: the lane's features' sums of g x over the tile's rows; g is zero for rows that do not
// count.  `bad`: rows left out that hold no numbers (0 x NaN is NaN), skipped.
//   columns: pairs of rows, g as [row pairs][classes][2]; the two sums of a pair meet at a flush
//   rows: pairs of features, g as [rows][classes][2 alike]
template <typename T, int C, bool COLS, int R, int F, int G = 1>
__device__ __forceinline__ void sums(Pair (&acc)[COLS ? F / 32 : F / 64][C], const uint8_t* tile, const float* g,
                                     uint32_t bad, int feats, int lane, int beside = 0) {
    using Geo = Tile<T, COLS, R, F, G>;
    constexpr int CL = padded<C>();
    if (COLS) {
        // lines lane + 32 f exchange alike; four rows of a line at a time
        const uint8_t* line = tile + lane * Geo::kLine;
        const int x0 = ((lane >> Geo::kShift) & Geo::kMask) << 4;
        constexpr int B = C <= 8 ? C : 4;                     // classes at a time
        // plain: numbers alone, no checks; features past the table give sums that nothing reads
        auto pass = [&](auto plain) {
            #pragma unroll
            for (int c0 = 0; c0 < C; c0 += B) {
                #pragma unroll 2
                for (int r = 0; r < R; r += 4) {
                    Pair g0[B], g1[B];
                    load_pairs<B>(g0, g + (r / 2 * CL + c0) * 2);
                    load_pairs<B>(g1, g + ((r / 2 + 1) * CL + c0) * 2);
                    const int b = (beside * R + r) * (int)sizeof(T);
                    const uint8_t* p = line + (((b >> 4 << 4) ^ x0) + (b & 15));
                    #pragma unroll
                    for (int f = 0; f < F / 32; ++f) {
                        if (!plain() && 32 * f >= feats) break;
                        float xv[4];
                        load4(xv, p + 32 * f * Geo::kLine, T{});
                        if (!plain())
                            #pragma unroll
                            for (int v = 0; v < 4; ++v)
                                if ((bad >> (r + v)) & 1) xv[v] = 0.f;
                        const Pair a = pair(xv[0], xv[1]), b2 = pair(xv[2], xv[3]);
                        #pragma unroll
                        for (int c = 0; c < B; ++c) {
                            acc[f][c0 + c] = fma2(a, g0[c], acc[f][c0 + c]);
                            acc[f][c0 + c] = fma2(b2, g1[c], acc[f][c0 + c]);
                        }
                    }
                }
            }
        };
        // (from five classes on two copies of the loop cost more in registers than the checks)
        if (C <= 4 && bad == 0 && (F == 64 || 2 * feats > F))
            pass([] { return true; });
        else
            pass([] { return false; });
    } else {
        constexpr int N = F / 32;                             // neighbouring features of a lane
        const int b = N * lane * (int)sizeof(T);
        const int own = (b >> 4) << 4;
        const uint8_t* p = tile + (b & 15);
        auto pass = [&](auto plain) {
            #pragma unroll 8
            for (int r = 0; r < R; ++r) {
                if (!plain() && ((bad >> r) & 1)) continue;
                float xv[N];
                Pair gv[C];
                load_some(xv, p + r * Geo::kLine + (own ^ ((r & 7) << 4)), T{});
                load_pairs<C>(gv, g + r * CL * 2);
                #pragma unroll
                for (int f = 0; f < N; f += 2) {
                    const Pair x = pair(xv[f], xv[f + 1]);
                    #pragma unroll
                    for (int c = 0; c < C; ++c) acc[f / 2][c] = fma2(x, gv[c], acc[f / 2][c]);
                }
            }
        };
        if (bad == 0)
            pass([] { return true; });
        else
            pass([] { return false; });
    }
}

// C: classes the code has room for (a.c of them exist); GRAD: dw, dbias or dx wanted; F: features of
// a warp's tile; VEC: x in 16-byte copies (kernels of their own, for the registers); G: groups
// whose tiles lie side by side
template <typename T, int C, bool COLS, bool GRAD, bool DX, int F, bool VEC, int G>
__global__ void __launch_bounds__(few_threads(F, GRAD), few_warps(C, F, GRAD) * 32 / few_threads(F, GRAD)) xent_few_kernel(const FewArgs a) {
    constexpr int CL = padded<C>(), NF = GRAD ? F / 32 : 1;   // NF: features a lane sums in step 3
    constexpr int NP = !GRAD ? 1 : COLS ? NF : NF / 2;         // its sums: pairs over rows, or over features
    constexpr int GL = COLS ? CL : 2 * CL;                     // floats of a row of g
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int W = a.warps, group = warp / W, wg = warp - group * W;   // warp wg of its group
    const int R = a.rows;
    const int warps = W * a.groups;
    const int tile_bytes = R * F * (int)sizeof(T);
    const int gi = G > 1 ? group % G : 0;                 // among the G groups that share a tile
    uint8_t* tile = smem + (size_t)(G > 1 ? wg * G + group - gi : warp) * tile_bytes;
    float* ws = reinterpret_cast<float*>(smem + (size_t)warps * tile_bytes);   // w, [d_pad][CL] or [d_pad / 2][CL][2]
    float* gs = ws + (size_t)a.d_pad * CL + (size_t)warp * (GRAD ? kRowsMost * GL : 0);   // g, a warp's own
    float* red = ws + (size_t)a.d_pad * CL + (size_t)warps * (GRAD ? kRowsMost * GL : 0);   // [2][groups][W][C][32]
    double* bsum = reinterpret_cast<double*>(red + (W > 1 ? 2 * (size_t)warps * C * 32 : 0)) +
                   (size_t)group * C * 32;                                                  // bias: [C][32] a group

    for (int i = threadIdx.x; i < a.d_pad * CL; i += blockDim.x) {
        const int k = i / CL, c = i % CL;
        ws[COLS ? i : (k / 2 * CL + c) * 2 + (k & 1)] =
            c < a.c && k < a.d ? to_float(((const T*)a.w)[c * a.wr + k * a.wk]) : 0.f;
    }
    float bias[C];
    #pragma unroll
    for (int c = 0; c < C; ++c) bias[c] = c < a.c ? (a.bias ? a.bias[c] : 0.f) : -INFINITY;
    if (GRAD && wg == 0)
        for (int c = 0; c < C; ++c) bsum[c * 32 + lane] = 0.0;
    __syncthreads();

    Pair acc[NP][C];
    float db[C];
    #pragma unroll
    for (int f = 0; f < NP; ++f)
        #pragma unroll
        for (int c = 0; c < C; ++c) acc[f][c] = 0;
    #pragma unroll
    for (int c = 0; c < C; ++c) db[c] = 0.f;

    const int row = R == 32   ? Lanes<COLS, 32>::row(lane)
                    : R == 16 ? Lanes<COLS, 16>::row(lane)
                              : Lanes<COLS, 8>::row(lane);
    const int share = lane >> a.log_rows, shares = 32 >> a.log_rows;   // among the lanes with this row
    const int kw = wg * F;                      // GRAD: the warp's features
    // The groups of a CTA take neighbouring tiles (of a wide table's columns they then read the
    // same pages); where there are few tiles, one group of every CTA comes first.
    const int64_t step = (int64_t)a.groups * gridDim.x;
    const int64_t first = G > 1 || a.n_tiles >= step ? (int64_t)blockIdx.x * a.groups + group
                                                     : (int64_t)group * gridDim.x + blockIdx.x;
    const size_t part_at = (size_t)first * a.c * a.d_pad;
    int parity = 0, since = 0;
    bool flushed = false;

    // sums so far to the group's partial
    auto flush = [&]() {
        if (a.part) {
            // several loads under way before their stores
            constexpr int B = NP * C <= 16 ? NP : 1, V = COLS ? 1 : 2;
            float* p = a.part + part_at + kw + (COLS ? lane : NF * lane);
            #pragma unroll
            for (int f0 = 0; f0 < NP; f0 += B) {
                float old[B][C][V] = {};
                if (flushed)
                    #pragma unroll
                    for (int f = 0; f < B; ++f)
                        #pragma unroll
                        for (int c = 0; c < C; ++c)
                            #pragma unroll
                            for (int v = 0; v < V; ++v)
                                if (c < a.c) old[f][c][v] = p[(size_t)c * a.d_pad + (COLS ? 32 : 2) * (f0 + f) + v];
                #pragma unroll
                for (int f = 0; f < B; ++f)
                    #pragma unroll
                    for (int c = 0; c < C; ++c) {
                        float lo, hi;
                        unpair(lo, hi, acc[f0 + f][c]);
                        acc[f0 + f][c] = 0;
                        if (c >= a.c) continue;
                        float* q = p + (size_t)c * a.d_pad + (COLS ? 32 : 2) * (f0 + f);
                        q[0] = old[f][c][0] + (COLS ? lo + hi : lo);
                        if (!COLS) q[V - 1] = old[f][c][V - 1] + hi;
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

    // The warp's tiles in order: with gradients one of every tile of rows, else all features of a
    // tile of rows in turn.
    const int k_first = GRAD ? kw : 0, k_step = GRAD ? a.d_pad : F;
    auto load = [&](int64_t t, int k0) {
        if (R == 32)
            load_tile<T, COLS, 32, F, VEC>(a, tile, t * R, k0, lane);
        else if (R == 16)
            load_tile<T, COLS, 16, F, VEC>(a, tile, t * R, k0, lane);
        else
            load_tile<T, COLS, 8, F, VEC>(a, tile, t * R, k0, lane);
    };
    // the warps of the groups that share a tile wait for each other (without gradients, two sets)
    auto together = [&]() {
        if (GRAD)
            __syncthreads();
        else if (group < G)
            asm volatile("bar.sync 1, %0;" ::"n"(32 * G) : "memory");
        else
            asm volatile("bar.sync 2, %0;" ::"n"(32 * G) : "memory");
    };
    struct Meta {
        int64_t y;
        float weight;
    };
    auto meta_of = [&](int64_t t) {
        Meta m = {-1, 0.f};
        const int64_t gr = t * R + row;
        if (t < a.n_tiles && gr < a.n) {
            m.y = a.labels[gr];
            if (GRAD) m.weight = (a.weight ? a.weight[gr * a.weight_stride] : 1.f) * a.scale;
        }
        return m;
    };
    Meta meta = meta_of(first);
    // (side by side, the groups of a CTA go on together: rows past the table's end are zeros)
    for (int64_t t = first; G > 1 ? t - group < a.n_tiles : t < a.n_tiles; t += step) {
        const int64_t r0 = t * R, gr = r0 + row;
        float z[C];
        #pragma unroll
        for (int c = 0; c < C; ++c) z[c] = 0.f;
        Meta next = meta;
        for (int k0 = k_first; k0 < a.d; k0 += k_step) {
            if constexpr (G > 1) {
                together();                                // the tiles' last readers are done
                load_side_by_side<T, F, G>(a, tile, (t - gi) * R, k0, gi, lane);
            } else {
                __syncwarp();                              // the tile's last readers are done
                load(t, k0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (k0 == k_first) next = meta_of(t + step);
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if constexpr (G > 1)
                together();
            else
                __syncwarp();
            // 1. a lane is a row
            const int feats = min(F, a.d - k0);
            const float* wk = ws + (size_t)k0 * CL;                // k0 / 2 pairs of 2 CL
            if constexpr (G > 1)
                dots<T, C, COLS, 32, F, G>(z, tile, wk, feats, lane, gi);
            else if (R == 32)
                dots<T, C, COLS, 32, F>(z, tile, wk, feats, lane);
            else if (R == 16)
                dots<T, C, COLS, 16, F>(z, tile, wk, feats, lane);
            else
                dots<T, C, COLS, 8, F>(z, tile, wk, feats, lane);
        }
        const int64_t y64 = meta.y;
        const float rw = meta.weight;
        meta = next;
        // 2. logits of all warps, softmax, loss, g
        if (GRAD && W > 1) {
            float* mine = red + ((size_t)(parity * a.groups + group) * W) * C * 32;
            #pragma unroll
            for (int c = 0; c < C; ++c) mine[(wg * C + c) * 32 + lane] = z[c];
            // (two groups at most; a barrier named by a register would reserve all 16, and an SM has
            // those of four CTAs)
            if (group)
                asm volatile("bar.sync 2, %0;" ::"r"(W * 32) : "memory");
            else
                asm volatile("bar.sync 1, %0;" ::"r"(W * 32) : "memory");
            #pragma unroll
            for (int c = 0; c < C; ++c) z[c] = 0.f;
            #pragma unroll 2
            for (int w = 0; w < W; ++w)
                #pragma unroll
                for (int c = 0; c < C; ++c) z[c] += mine[(w * C + c) * 32 + lane];
            parity ^= 1;
        }
        const bool kept = y64 >= 0;
        const int y = kept && y64 < a.c ? (int)y64 : -1;   // kept with y < 0: no such class
        const bool finite = fabsf(z[0]) <= 3.402823466e38f;   // any NaN or infinity in the row shows here
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
            // e / s, whether the loss is there or not: logits far from zero leave a given lse, rounded
            // to its last bit, too coarse for exp(z - lse)
            const float inv = 1.f / s;
            // bit r: row r is left out and holds something that is no number
            uint32_t bad = 0;
            if (__any_sync(0xffffffffu, !kept && !finite)) bad = __reduce_or_sync(0xffffffffu, !kept && !finite ? 1u << row : 0u);
            #pragma unroll
            for (int c = 0; c < C; ++c) {
                float g = kept ? (e[c] * inv - (c == y ? 1.f : 0.f)) * rw : 0.f;
                if (kept && y < 0) g = NAN;
                if (c >= a.c) g = 0.f;
                e[c] = g;
                if (share == 0) {
                    if (COLS)
                        gs[(row / 2 * CL + c) * 2 + (row & 1)] = g;
                    else
                        *reinterpret_cast<Pair*>(gs + (row * CL + c) * 2) = pair(g, g);
                    db[c] += g;
                }
            }
            __syncwarp();
            if (DX) {
                const int left = (int)min((int64_t)R, a.n - r0), feats = min(F, a.d - kw);
                T* dx = (T*)a.dx + r0 * a.dxr + (int64_t)kw * a.dxk;
                const uint32_t rows_in = COLS ? 0 : __reduce_or_sync(0xffffffffu, kept ? 1u << row : 0u);   // rows that count
                const float* wk = ws + (size_t)kw * CL;
                if (COLS) {
                    // neighbouring lanes are neighbouring rows
                    if (row < left)
                        #pragma unroll 4
                        for (int k = share; k < feats; k += shares) {
                            float v = 0.f;
                            #pragma unroll
                            for (int c = 0; c < C; ++c) v = fmaf(e[c], wk[k * CL + c], v);
                            dx[row * a.dxr + k * a.dxk] = from_float<T>(kept ? v : 0.f);
                        }
                } else {
                    for (int k = lane; k < feats; k += 32) {
                        float wv[C];
                        #pragma unroll
                        for (int c = 0; c < C; ++c) wv[c] = wk[(k / 2 * CL + c) * 2 + (k & 1)];
                        #pragma unroll 4
                        for (int r = 0; r < left; ++r) {
                            float v = 0.f;
                            #pragma unroll
                            for (int c = 0; c < C; ++c) v = fmaf(gs[(r * CL + c) * 2], wv[c], v);
                            dx[r * a.dxr + k * a.dxk] = from_float<T>((rows_in >> r) & 1 ? v : 0.f);
                        }
                    }
                }
            }
            // 3. a lane is two or four features
            if constexpr (GRAD) {
                if (a.part && __any_sync(0xffffffffu, kept)) {
                    const int feats = min(F, a.d - kw);
                    if constexpr (G > 1)
                        sums<T, C, COLS, 32, F, G>(acc, tile, gs, bad, feats, lane, gi);
                    else if (R == 32)
                        sums<T, C, COLS, 32, F>(acc, tile, gs, bad, feats, lane);
                    else if (R == 16)
                        sums<T, C, COLS, 16, F>(acc, tile, gs, bad, feats, lane);
                    else
                        sums<T, C, COLS, 8, F>(acc, tile, gs, bad, feats, lane);
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

template <typename T, int C, bool COLS, bool GRAD, bool DX, int F, bool VEC, int G>
cudaError_t launch_f(const FewPlan& p, cudaStream_t stream) {
    auto fn = xent_few_kernel<T, C, COLS, GRAD, DX, F, VEC, G>;
    static SharedMemory shared;
    const cudaError_t e = shared.allow((const void*)fn, kFewMaxSmem);
    if (e != cudaSuccess) return e;
    KernelTimer kt(stream, GAFIME_KERNEL_XENT);
    fn<<<p.grid, p.threads, p.smem, stream>>>(p.k);
    return cudaGetLastError();
}

template <typename T, int C, bool COLS, bool GRAD, bool DX, int F>
cudaError_t launch_g(const FewPlan& p, cudaStream_t s) {
    if constexpr (COLS && (GRAD || C <= kBesideMaxC)) {
        if (p.beside == 4) return launch_f<T, C, COLS, GRAD, DX, F, true, 4>(p, s);
        if constexpr (GRAD && F == 128)
            if (p.beside == 2) return launch_f<T, C, COLS, GRAD, DX, F, true, 2>(p, s);
    }
    return p.vec ? launch_f<T, C, COLS, GRAD, DX, F, true, 1>(p, s) : launch_f<T, C, COLS, GRAD, DX, F, false, 1>(p, s);
}

template <typename T, int C, bool COLS, bool GRAD, bool DX>
cudaError_t launch(const FewPlan& p, cudaStream_t s) {
    if constexpr (GRAD)
        if (p.features == 128) return launch_g<T, C, COLS, GRAD, DX, 128>(p, s);
    return launch_g<T, C, COLS, GRAD, DX, 64>(p, s);
}

template <typename T, int C, bool COLS>
cudaError_t launch_c(const FewPlan& p, cudaStream_t s) {
    if (!p.grad) return launch<T, C, COLS, false, false>(p, s);
    if constexpr (C <= kFewMaxGrad)
        return p.k.dx ? launch<T, C, COLS, true, true>(p, s) : launch<T, C, COLS, true, false>(p, s);
    return cudaErrorInvalidValue;
}

template <typename T, bool COLS>
cudaError_t launch_t(const FewPlan& p, cudaStream_t s) {
    switch (p.cp) {
        case 2: return launch_c<T, 2, COLS>(p, s);
        case 3: return launch_c<T, 3, COLS>(p, s);
        case 4: return launch_c<T, 4, COLS>(p, s);
        case 6: return launch_c<T, 6, COLS>(p, s);
        case 8: return launch_c<T, 8, COLS>(p, s);
        case 16: return launch_c<T, 16, COLS>(p, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace few

}  // namespace gafime
