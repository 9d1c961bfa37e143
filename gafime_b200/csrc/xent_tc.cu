// xent_tc.cu -- softmax cross entropy of a linear head with many classes, on the tensor cores.
//
// The n x c logits never exist as a whole.  A forward call forms 256 x BN tiles of them in tensor
// memory and keeps, per row, the running maximum and sum of exponentials.  A gradient call forms
// them again piece by piece (piece_bytes at a time), writes a piece's
//   g_ij = r_i (exp(z_ij - lse_i) - [j = y(i)])
// in 16 bits and multiplies it with both sides:
//   lse   z = x w^T, online softmax in the epilogue              2 n d c FLOP
//   g     z again, g in the epilogue                             2 n d c
//   both  where one tile holds every class (256 and fewer): loss and g from the same z
//   dx    g w        (classes summed; fp32 sums kept between class pieces)
//   dw    g^T x      (rows summed; split over rows where the c x d tiles are few)
//
// Types.  16-bit x and w are multiplied as they are (TMA reads them in place where their
// strides allow, else from a copy); g is rounded once to their type (half a step, 2^-8 or 2^-11
// relative, independent from element to element, which is what rounding the result costs too); in
// fp16 it is scaled by a power of two first, from the largest row weight, and held to 2^-38 of that:
// fp16's own 40 bits, from the largest row's gradients down to steps that its outputs have as well.
// An fp32 value is held as three bf16 planes, its bits eight by eight, x = h + m + l exactly
// (below 2^-110, to 2^-134), and so is g in fp32.  bf16 has fp32's exponents, so there is nothing to
// scale and no value changes another's bits: a row, a feature, a class or a row weight far above the
// others leaves them as they are.  A product is
//   l h + h l + m m + m h + h m + h h        (left out: m l, l m, l l, below 3 x 2^-23 of |x||w|)
// six 16-bit products, with everything that a 24-bit product holds but its last bit or two.  Two
// fp16 planes with common scales would take three, but hold only 38 bits below the largest value.
// A weight of +-infinity sits in a fourth plane of its own, which only x's h meets (its m and l have
// signs of their own, and 0 x inf is no number): a product more where there is such a weight.
//
// Kernel (pairs of CTAs, one CTA an SM, persistent, 12 warps; a pair makes 256 x BN tiles): warp 0
// queues its CTA's TMA loads of 128 x 64 of A and BN / 2 x 64 of B into a ring; warp 1 of the
// pair's first CTA issues the MMAs into one of two tensor-memory accumulators; warps 4-11 turn
// the other accumulator's 128 rows of their CTA into sums, g, dx or dw.  Every mbarrier wait is
// bounded; one that gives up records a code, and everything that the call writes becomes NaN.
//
// What bounds it, measured on a B200 (1,645 TFLOP/s bf16 in a burst, 1,381 sustained under the
// power cap):
//   16 bits, 8192 x 1024, 32768 classes (0.55 TFLOP a product): lse 0.41 ms, g 0.47, dx 0.45, dw
//     0.45 = 1,150 to 1,340 TFLOP/s, 83 to 97 % of the sustained rate.  With the MMAs left out the
//     loads alone take 0.29 ms; g adds its exponentials, packing, stores and column sums.
//   fp32, 200000 x 256, 1000 classes (6 products of 0.10 TFLOP): lse 0.45 ms, g 0.73, dx 0.50, dw
//     0.51 = 1,370 TFLOP/s of 16-bit products in lse, 1,230 in dx and dw: the tensor cores; g 850,
//     bound by its epilogue (exponentials, three planes, column sums).  Two scaled fp16 planes took
//     0.26, 0.43, 0.31 and 0.30 ms, and lost rows beside a large value.
// Pairs of CTAs against single ones of 128 x 256 (16 bits): lse 0.54 -> 0.41 ms together with even
// runs of class tiles, dw 0.47 -> 0.45.  Pieces of half the size: dx nearly twice as long (one round
// of the pairs to a launch exposes its start and end); of 256 MB in place of 384 with three planes,
// the step of 8192 x 1024 with 8192 classes 1.71 -> 2.37 ms.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <iterator>
#include <mutex>
#include <type_traits>

#include "engine.h"
#include "tc.cuh"
#include "xent.h"

namespace gafime {

namespace {

constexpr int kThreads = 384;
// Registers: 384 x 168 at launch = 128 x 40 (loads, MMAs) + 256 x 232 (epilogues, which keep a
// tile's 128 sums a thread)
constexpr int kControlRegs = 40, kEpiRegs = 232;
static_assert(128 * kControlRegs + 256 * kEpiRegs <= kThreads * 168, "registers of the launch");
constexpr int kEpiWarps = 8;
constexpr int kBM = 128;                     // rows of a CTA's half of a tile
constexpr int kPM = 256;                     // rows of a pair's tile
constexpr int kBK = 64;                      // 16-bit values of K to a stage
constexpr int kABytes = kBM * kBK * 2;
constexpr float kLog2e = 1.4426950408889634f;
// Of a piece of g: several rounds of the pairs, not the n x c whole.  Three planes get as many values
// as two would in 256 MB.
constexpr size_t piece_bytes(int planes) { return (size_t)(planes == 3 ? 384 : 256) << 20; }

enum { LSE = 0, G = 1, DX = 2, DW = 3, BOTH = 4 };

constexpr int stage_bytes(int bn) { return kABytes + bn / 2 * kBK * 2; }   // of one CTA
// Ring stages.  fp32 holds three of them for a block of K and hands the first back a third of the
// way through its products, so four keep the next block's loads under way.
constexpr int stages_of(int bn, int out) { return bn == 256 ? (out > 4096 ? 4 : 6) : bn == 128 ? (out > 4096 ? 5 : 8) : out > 4096 ? 6 : 8; }
// An epilogue warp's outgoing blocks: 32 rows x 128 bytes of each plane of g (64 bytes where a tile
// has 64 columns), or of dx or dw (64 bytes in 16 bits).
constexpr int out_bytes(int mode, int planes) { return (mode == G || mode == BOTH) && planes == 3 ? 12288 : 4096; }
constexpr size_t smem_of(int bn, int out) {
    return (size_t)stages_of(bn, out) * stage_bytes(bn) + kEpiWarps * out + 1024 + 256;
}
static_assert(smem_of(256, 4096) <= 232448 && smem_of(128, 4096) <= 232448 && smem_of(64, 4096) <= 232448 &&
                  smem_of(256, 12288) <= 232448 && smem_of(128, 12288) <= 232448 && smem_of(64, 12288) <= 232448,
              "shared memory per CTA");

// What the kernels of one call share on the device; cleared at its start.
struct Meta {
    int err;                 // code of a wait that gave up
    uint32_t weight_bits;    // largest finite |row weight| as float bits
    uint32_t far;            // a given lse is too coarse to normalise with
    uint32_t wild;           // fp32: some weight is infinite
    uint32_t poison;         // some left-out row of an x read in place holds a value that is not finite
};

// exponent that brings a largest magnitude below 2^14 (0 for nothing to bring)
__device__ __forceinline__ int fit_exponent(uint32_t max_bits) {
    if (max_bits == 0) return 0;
    const int e = (int)(max_bits >> 23) - 127;
    return min(126, max(-126, 13 - e));
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // -126 .. 127
// v 2^e for any e that two factors reach
__device__ __forceinline__ float scale2(float v, int e) {
    e = min(252, max(-252, e));
    const int h = e / 2;
    return v * pow2i(h) * pow2i(e - h);
}
// e^v; below 2^-126 zero, which is nothing beside the sums it enters (2^-22 relative otherwise, and
// 2^-24 |v|).  Logits stay in base e up to the difference that comes here: one of the type's lowest
// value, a mask's, has no finite double in base 2.
__device__ __forceinline__ float exp_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * kLog2e));
    return r;
}
__device__ __forceinline__ int g_exponent(const Meta* m, int half_g) { return half_g ? fit_exponent(m->weight_bits) : 0; }

struct TcArgs {
    CUtensorMap a[3], b[4];   // planes: one, or h, m, l of fp32, w's infinities (b[1] also: see cleaned)
    CUtensorMap out[3];       // G: planes of g; DX, DW: dx, dw
    int if_far;               // LSE: nothing to do unless meta->far is set
    int half_g;               // g in fp16 (scaled by 2^u), else bf16
    int units, m_tiles, n_tiles, splits;
    int per_split;            // LSE: class tiles of a split; DW: k blocks of a split
    int k_blocks;
    int chunk;                // k blocks summed in tensor memory at a time
    int a_row0, b_row0;       // first row of the piece in the maps of x; of the class piece in that of w
    int64_t rows;             // valid rows (LSE, G, DX: of x or the piece), DW: classes
    int64_t row0;             // the piece's first row in labels, loss, dx
    int64_t cols;             // valid columns: LSE, G: classes (of the piece); DX, DW: features
    int64_t c_total;
    int c0;                   // first class of the piece
    Meta* meta;
    const float* bias;        // -inf past the classes
    const int64_t* labels;
    float *loss_out, *lse_out;   // BOTH: [n]; null: not wanted
    float2* part;             // LSE: [n][2 splits] maximum, sum
    float* zy;                // LSE: label's logit
    const float2* shift;      // G: [n] maximum and log of the sum
    const float* loss;        // G
    const float* weight;
    int64_t weight_stride;
    float scale;
    int64_t ldg;              // G: columns of its planes
    float* bias_part;         // G: sums of 32 rows, [row tile x 4][ldg]; null: not wanted
    void* dx;                 // DX; DW: dw
    int64_t dxr, dxk;
    int dx_map;               // out[0] is valid; else element stores
    int first, last;          // DX: first / last class piece; DW: first / last row piece
    float* sums;              // DX, DW: [split][128-row tile][feature tile][BN][128] of pieces and splits
    int64_t split_stride;
    int64_t tile0;            // DW: first tile of the class piece
    int direct;               // one split, whose last piece leaves as dx or dw
    int cleaned;              // DW: b[1] is a copy of x without such rows, there when meta->poison is set
};

__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The bf16 thirds of two fp32 values, a in the lower halves: h the upper 8 bits, cut (rounding could
// leave the type), m the next 8 of what is left, rounded, and l the rest.
__device__ __forceinline__ void thirds(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    h = __byte_perm(ua, ub, 0x7632);
    const float ra = a - __uint_as_float(ua & 0xffff0000u), rb = b - __uint_as_float(ub & 0xffff0000u);
    m = pack(ra, rb, __nv_bfloat16{});
    l = pack(ra - __uint_as_float(m << 16), rb - __uint_as_float(m & 0xffff0000u), __nv_bfloat16{});
}

// Outgoing blocks of 32 rows (the lanes) x 32 columns in shared memory, as TMA stores read them:
// 16-byte units of a row exchanged by the 64-byte (16 bits) or 128-byte (fp32) swizzle, which
// also spreads the lanes' writes over the banks.
template <typename T>
__device__ __forceinline__ int out_unit(int row, int q) {
    return sizeof(T) == 4 ? row * 128 + ((q ^ (row & 7)) << 4) : row * 64 + ((q ^ ((row >> 1) & 3)) << 4);
}
template <typename T>
__device__ __forceinline__ void out_write(uint8_t* block, int row, const float* v) {
    constexpr int V = 16 / sizeof(T);
    #pragma unroll
    for (int q = 0; q < 32 / V; ++q) {
        uint4 u;
        if constexpr (sizeof(T) == 4)
            u = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                           __float_as_uint(v[4 * q + 3]));
        else
            u = make_uint4(pack(v[8 * q], v[8 * q + 1], T{}), pack(v[8 * q + 2], v[8 * q + 3], T{}),
                           pack(v[8 * q + 4], v[8 * q + 5], T{}), pack(v[8 * q + 6], v[8 * q + 7], T{}));
        *reinterpret_cast<uint4*>(block + out_unit<T>(row, q)) = u;
    }
}
// the same of g's blocks, SPAN x 32 columns of 16 bits
template <int SPAN>
__device__ __forceinline__ int g_unit(int row, int q) {
    return SPAN == 2 ? row * 128 + ((q ^ (row & 7)) << 4) : row * 64 + ((q ^ ((row >> 1) & 3)) << 4);
}
template <typename T>
__device__ __forceinline__ T* out_at(uint8_t* block, int row, int col) {
    constexpr int V = 16 / sizeof(T);
    return reinterpret_cast<T*>(block + out_unit<T>(row, col / V)) + col % V;
}

// A unit of work: `tiles` accumulator tiles (m, n), (m, n + 1), ... (more than one only in LSE),
// each over the k blocks [kb, kb + kn), a.chunk of them at a time in tensor memory.
struct Unit {
    int m, n, split, tiles, kb, kn;
};
template <int MODE>
__device__ __forceinline__ Unit unit_of(const TcArgs& a, int u) {
    Unit t;
    t.split = 0;
    t.tiles = 1;
    t.kb = 0;
    t.kn = a.k_blocks;
    if (MODE == LSE) {
        t.m = u % a.m_tiles;
        t.split = u / a.m_tiles;
        t.n = t.split * a.per_split;
        t.tiles = min(a.per_split, a.n_tiles - t.n);
    } else if (MODE == G || MODE == BOTH) {
        t.m = u % a.m_tiles;
        t.n = u / a.m_tiles;
    } else {
        const int tiles = a.m_tiles * a.n_tiles, tile = u % tiles;
        t.split = u / tiles;
        t.n = tile % a.n_tiles;
        t.m = tile / a.n_tiles;
        t.kb = t.split * a.per_split;
        t.kn = max(0, min(a.per_split, a.k_blocks - t.kb));
    }
    return t;
}

// Sums over the warp's lanes of 32 values each: lane j gets the sum of everyone's v[j].  Each
// step halves what a lane holds: 31 shuffles in place of 32 x 5.
__device__ __forceinline__ float column_sums(float* v, int lane) {
    #pragma unroll
    for (int o = 16; o; o >>= 1) {
        const bool upper = lane & o;
        #pragma unroll
        for (int j = 0; j < o; ++j) {
            const float send = upper ? v[j] : v[j + o], keep = upper ? v[j + o] : v[j];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    return v[0];
}

// v[i] for a run-time i in [0, 32): a select tree
__device__ __forceinline__ float pick(const float* v, int i) {
    float t[16];
    #pragma unroll
    for (int j = 0; j < 16; ++j) t[j] = i & 16 ? v[j + 16] : v[j];
    #pragma unroll
    for (int o = 8; o; o >>= 1)
        #pragma unroll
        for (int j = 0; j < o; ++j) t[j] = i & o ? t[j + o] : t[j];
    return t[0];
}

// E: type of the operand planes; kPlanes: 1, or the three of fp32
template <int MODE, int BN, typename E, int kPlanes>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) xent_tc_kernel(const __grid_constant__ TcArgs a) {
    constexpr int kOut = out_bytes(MODE, kPlanes);
    constexpr int S = stages_of(BN, kOut), kCols = BN / 2;   // ring stages; columns of an epilogue thread
    constexpr bool kG = MODE == G || MODE == BOTH, kZ = kG || MODE == LSE;
    constexpr bool kAMn = MODE == DW, kBMn = MODE == DX || MODE == DW;
    constexpr bool kBf16 = sizeof(E) == 2 && !std::is_same<E, __half>::value;
    constexpr uint32_t kId = tc::idesc(BN, kBf16, kAMn, kBMn);
    if (MODE == LSE && a.if_far && a.meta->far == 0) return;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (tc::smem_addr(raw) + 1023) & ~1023u;
    uint8_t* gbase = raw + (base - tc::smem_addr(raw));
    const uint32_t outs = base + S * stage_bytes(BN);         // a multiple of 1024
    const uint32_t bars = outs + kEpiWarps * kOut;
    const uint32_t full0 = bars, empty0 = bars + 8 * S, afull0 = bars + 16 * S, aempty0 = afull0 + 16,
                   drain = afull0 + 32, slot = afull0 + 40;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)tc::cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    int* err = &a.meta->err;
    const bool wild = kPlanes == 3 && MODE != DW && a.meta->wild != 0;
    const int stages = kPlanes + wild;                        // of a block of K

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::bar_init(full0 + 8 * s, 1);
            tc::bar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc::bar_init(afull0 + 8 * s, 1);
            tc::bar_init(aempty0 + 8 * s, 2 * kEpiWarps);   // of both CTAs, in the leader
        }
        tc::bar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tc::tmem_alloc(slot, 2 * BN);
    tc::fence_before();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + (slot - base));

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == 0) {
            // ---- loads
            if (lane == 0) {
                uint32_t k = 0;   // stages handed out
                bool ok = true;
                const bool clean = MODE == DW && a.cleaned && a.meta->poison != 0;
                const uint32_t full_l = tc::in_leader(full0);
                for (int u = pair; ok && u < a.units; u += pairs) {
                    const Unit t = unit_of<MODE>(a, u);
                    const int m0 = t.m * kPM + rank * kBM;
                    for (int r = 0; ok && r < t.tiles; ++r) {
                        const int n0 = (t.n + r) * BN + rank * (BN / 2);
                        // three planes: a block of K takes three stages, l, h and m of both sides, and
                        // where some weight is infinite a fourth, h and the infinities
                        for (int i = 0; i < t.kn * stages; ++i, ++k) {
                            const int kb = t.kb + i / stages, q = i % stages;
                            const int plane = kPlanes == 1 || q == 3 ? 0 : (q + 2) % 3;
                            const CUtensorMap* ma = &a.a[plane];
                            const CUtensorMap* mb = &a.b[clean ? 1 : q == 3 ? 3 : plane];
                            const uint32_t s = k % S, full = full_l + 8 * s;
                            // (a wait of a second is over long after the copies before it)
                            if (k >= S && !(ok = tc::bar_wait(empty0 + 8 * s, ((k / S) - 1) & 1, err, 1))) break;
                            if (rank == 0) tc::bar_expect(full0 + 8 * s, 2 * stage_bytes(BN));
                            const uint32_t sa = base + s * stage_bytes(BN), sb = sa + kABytes;
                            if (kAMn) {
                                tc::load_2d(sa, ma, full, m0, kb * kBK);
                                tc::load_2d(sa + kABytes / 2, ma, full, m0 + 64, kb * kBK);
                            } else {
                                tc::load_2d(sa, ma, full, kb * kBK, a.a_row0 + m0);
                            }
                            if (kBMn) {
                                #pragma unroll
                                for (int h = 0; h < BN / 128; ++h)
                                    tc::load_2d(sb + h * 8192, mb, full, n0 + h * 64, a.b_row0 + kb * kBK);
                            } else {
                                tc::load_2d(sb, mb, full, kb * kBK, a.b_row0 + n0);
                            }
                        }
                    }
                }
            }
        } else if (warp == 1 && rank == 0) {
            // ---- MMAs, for both CTAs
            uint32_t k = 0, acc = 0;
            bool ok = true;
            for (int u = pair; ok && u < a.units; u += pairs) {
                const Unit t = unit_of<MODE>(a, u);
                const int end = t.tiles * t.kn;
                for (int i = 0; ok && i < end;) {
                    // one chunk: the blocks up to a multiple of a.chunk or the tile's end
                    const int in_tile = i % t.kn, stop = i + min(a.chunk, t.kn - in_tile);
                    const uint32_t d = tmem + (acc & 1) * BN;
                    if (acc >= 2 && !(ok = tc::bar_wait_warp(aempty0 + 8 * (acc & 1), ((acc >> 1) - 1) & 1, err, 3))) break;
                    tc::fence_after();
                    bool more = false;
                    auto multiply = [&](uint32_t sa, uint32_t sb) {   // stages of A and of B
                        const uint64_t da = tc::desc(base + sa * stage_bytes(BN), kAMn);
                        const uint64_t db = tc::desc(base + sb * stage_bytes(BN) + kABytes, kBMn);
                        #pragma unroll
                        for (int j = 0; j < kBK / 16; ++j) {
                            tc::mma(d, da + j * (kAMn ? 2048 >> 4 : 32 >> 4), db + j * (kBMn ? 2048 >> 4 : 32 >> 4), kId, more);
                            more = true;
                        }
                    };
                    if constexpr (kPlanes == 1) {
                        for (; i < stop; ++i, ++k) {
                            const uint32_t s = k % S;
                            if (!(ok = tc::bar_wait_warp(full0 + 8 * s, (k / S) & 1, err, 4))) break;
                            tc::fence_after();
                            if (lane == 0) {
                                multiply(s, s);
                                tc::commit_both(empty0 + 8 * s);
                            }
                            __syncwarp();
                        }
                    } else {
                        // (one block of K to a chunk) the small products first, as the stages arrive: what
                        // the tensor cores cut off is a part of the sum so far
                        for (; i < stop; ++i, k += stages) {
                            const uint32_t sl = k % S, sh = (k + 1) % S, sm = (k + 2) % S, si = (k + 3) % S;
                            auto arrived = [&](uint32_t q) {
                                ok = ok && tc::bar_wait_warp(full0 + 8 * (q % S), (q / S) & 1, err, 4);
                                return ok;
                            };
                            if (!arrived(k) || !arrived(k + 1)) break;
                            tc::fence_after();
                            if (lane == 0) {
                                multiply(sl, sh);
                                multiply(sh, sl);
                                tc::commit_both(empty0 + 8 * sl);
                            }
                            __syncwarp();
                            if (!arrived(k + 2) || (wild && !arrived(k + 3))) break;
                            tc::fence_after();
                            if (lane == 0) {
                                multiply(sm, sm);
                                multiply(sm, sh);
                                multiply(sh, sm);
                                tc::commit_both(empty0 + 8 * sm);
                                if (wild) {
                                    multiply(si, si);
                                    tc::commit_both(empty0 + 8 * si);
                                }
                                multiply(sh, sh);
                                tc::commit_both(empty0 + 8 * sh);
                            }
                            __syncwarp();
                        }
                    }
                    if (ok && lane == 0) tc::commit_both(afull0 + 8 * (acc & 1));
                    ++acc;
                    __syncwarp();
                }
            }
            // what was issued ends before the tensor memory is handed back
            if (lane == 0) {
                tc::commit(drain);
                tc::bar_wait(drain, 0, err, 5);
            }
            __syncwarp();
        }
    } else {
        // ---- epilogues
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const uint32_t out_addr = outs + (warp - 4) * kOut;
        uint8_t* out = gbase + (out_addr - base);
        uint32_t acc = 0;
        bool ok = true;
        const int ue = g_exponent(a.meta, a.half_g);
        const uint32_t aempty_l = tc::in_leader(aempty0);
        // What a unit needs of its rows is loaded while the unit before it is worked on.
        struct Row {
            int64_t y;
            float weight, loss;
            float2 shift;
        };
        auto row_of = [&](int u) {
            Row r = {-1, 1.f, 0.f, make_float2(0.f, 0.f)};
            if (MODE == DW || u >= a.units) return r;
            const int64_t row = (int64_t)(2 * unit_of<MODE>(a, u).m + rank) * kBM + quarter * 32 + lane;
            if (row >= a.rows) return r;
            r.y = a.labels[a.row0 + row];
            if (kG && a.weight) r.weight = a.weight[(a.row0 + row) * a.weight_stride];
            if (MODE == G) {
                r.loss = a.loss[a.row0 + row];
                r.shift = a.shift[a.row0 + row];
            }
            return r;
        };
        Row next = row_of(pair);
        for (int u = pair; ok && u < a.units; u += pairs) {
            const Unit t = unit_of<MODE>(a, u);
            const Row own_row = next;
            next = row_of(u + pairs);
            const int mt = 2 * t.m + rank;                 // this CTA's 128 rows
            const int64_t y0 = (int64_t)mt * kBM + quarter * 32, row = y0 + lane;
            const bool valid = row < a.rows;
            int64_t y = -1;
            float top = -INFINITY, sum = 0.f, zy = NAN;    // LSE
            float2 sh = make_float2(0.f, 0.f);             // G
            float wt = 0.f, ws = 0.f, gy = 0.f;            // G: ws the weight over the row's sum
            if (MODE != DW) y = own_row.y;
            if (kG && y >= 0) {
                wt = scale2(own_row.weight * a.scale, ue);
                if (y >= a.c_total) wt = NAN;
                if (MODE == G) {
                    sh = own_row.shift;
                    // exp(z_y - lse) - 1 from the loss, without the cancellation
                    gy = expm1f(-own_row.loss) * wt;
                    ws = wt * expf(-sh.y);
                }
            }
            for (int r = 0; ok && r < t.tiles && t.kn > 0; ++r) {
                const int n = t.n + r;
                // the tile's sums: chunks are added here, rounded to nearest (the tensor cores cut
                // what falls below an accumulator's last bit, so a long sum there drifts)
                float sums[kCols];
                #pragma unroll
                for (int j = 0; j < kCols; ++j) sums[j] = 0.f;
                for (int kb = 0; ok && kb < t.kn; kb += a.chunk, ++acc) {
                    if (!(ok = tc::bar_wait_warp(afull0 + 8 * (acc & 1), (acc >> 1) & 1, err, 6))) break;
                    tc::fence_after();
                    #pragma unroll
                    for (int ch = 0; ch < kCols / 32; ch += 2) {
                        // two loads under way before the wait
                        float v[32], w[32];
                        const uint32_t at = tmem + (acc & 1) * BN + half * kCols + ch * 32 + lane_addr;
                        tc::tmem_load32(at, v);
                        if constexpr (kCols > 32) tc::tmem_load32(at + 32, w);
                        tc::tmem_wait(v);
                        if constexpr (kCols > 32) tc::tmem_settle(w);
                        if (ch + 2 >= kCols / 32) {
                            tc::fence_before();
                            __syncwarp();
                            if (lane == 0) tc::bar_arrive_cluster(aempty_l + 8 * (acc & 1));
                        }
                        #pragma unroll
                        for (int j = 0; j < 32; ++j) sums[ch * 32 + j] += v[j];
                        if constexpr (kCols > 32)
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) sums[ch * 32 + 32 + j] += w[j];
                    }
                }
                if constexpr (MODE == BOTH) {
                    // the row's maximum and sum over this half's classes, its exponentials left in sums
                    const int blocks = (int)min((int64_t)(kCols / 32), max((int64_t)0, (a.cols - half * kCols + 31) / 32));
                    float m4[4] = {top, top, top, top};
                    #pragma unroll
                    for (int ch = 0; ch < kCols / 32; ++ch) {
                        if (ch >= blocks) break;
                        float* v = sums + ch * 32;
                        const int cb = half * kCols + ch * 32;
                        const float4* b4 = reinterpret_cast<const float4*>(a.bias + cb);
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 b = __ldg(b4 + j);
                            v[4 * j] += b.x;
                            v[4 * j + 1] += b.y;
                            v[4 * j + 2] += b.z;
                            v[4 * j + 3] += b.w;
                        }
                        #pragma unroll
                        for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], v[j]);
                        const int64_t rel = y - cb;
                        const bool here = rel >= 0 && rel < 32 && y < a.c_total;
                        if (__any_sync(0xffffffffu, here)) {
                            const float q = pick(v, (int)rel & 31);
                            if (here) zy = q;
                        }
                    }
                    top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    const float own = top == -INFINITY ? 0.f : top;   // nothing but excluded classes
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
                    #pragma unroll
                    for (int ch = 0; ch < kCols / 32; ++ch) {
                        if (ch >= blocks) break;
                        float* v = sums + ch * 32;
                        #pragma unroll
                        for (int j = 0; j < 32; ++j) s4[j & 3] += v[j] = exp_fast(v[j] - own);
                    }
                    sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    // and over the other half's, from the warp that has it.  A warp whose wait gave up
                    // comes here too, so that neither waits for good.
                    tc::store_wait_read<0>();          // the last store has read the block
                    reinterpret_cast<float4*>(out)[lane] = make_float4(top, sum, zy, ok ? 1.f : 0.f);
                    asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");
                    const float4 o = reinterpret_cast<const float4*>(out + (half ? -4 : 4) * kOut)[lane];
                    asm volatile("bar.sync %0, 64;" ::"r"(quarter + 1) : "memory");   // read before g is written there
                    ok = ok && o.w != 0.f;
                    const float m = fmaxf(top, o.x), shift = m == -INFINITY ? 0.f : m;
                    const float l = logf(sum * expf(top - shift) + o.y * expf(o.x - shift));
                    if (isnan(zy)) zy = o.z;
                    const float loss = y >= 0 ? (shift - zy) + l : 0.f;
                    if (half == 0 && valid && a.loss_out) {
                        a.loss_out[a.row0 + row] = loss;
                        if (a.lse_out)
                            a.lse_out[a.row0 + row] = y >= 0 ? shift + l : 0.f;
                    }
                    gy = expm1f(-loss) * wt;
                    // (with no class of its own a half's exponentials are zeros, whatever their shift)
                    ws = wt * (top == -INFINITY ? 0.f : expf((own - shift) - l));
                }
                if (!ok) break;
                #pragma unroll
                for (int ch = 0; ch < kCols / 32; ++ch) {
                    const int col = half * kCols + ch * 32;
                    const int64_t cb = (int64_t)n * BN + col;         // column of the piece
                    if (cb >= a.cols) break;
                    float* v = sums + ch * 32;
                    if (MODE == LSE || MODE == G) {   // (BOTH: done)
                        const float4* b4 = reinterpret_cast<const float4*>(a.bias + a.c0 + cb);
                        #pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 b = __ldg(b4 + j);
                            v[4 * j] += b.x;
                            v[4 * j + 1] += b.y;
                            v[4 * j + 2] += b.z;
                            v[4 * j + 3] += b.w;
                        }
                    }
                    // the row's label among these columns
                    const int64_t rel = y - a.c0 - cb;
                    const bool here = kZ && rel >= 0 && rel < 32 && y < a.c_total;
                    uint32_t hit = 0;
                    if (kZ) hit = __ballot_sync(0xffffffffu, here);
                    if (MODE == LSE) {
                        if (hit) {
                            const float q = pick(v, (int)rel & 31);
                            if (here) zy = q;
                        }
                    } else if (kG) {
                        #pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float p = (MODE == BOTH ? v[j] : exp_fast(v[j] - sh.x)) * ws;
                            v[j] = y >= 0 ? p : 0.f;
                        }
                        // 64 columns a store where the thread has as many: whole 128-byte lines
                        constexpr int kSpan = kCols >= 64 ? 2 : 1;       // blocks of 32 columns in one
                        constexpr int kPlane = 2048 * kSpan;
                        const int q0 = (ch % kSpan) * 4;
                        if (q0 == 0) tc::store_wait_read<0>();          // the last store has read them
                        #pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint8_t* to = out + g_unit<kSpan>(lane, q0 + q);
                            uint32_t h[4], m[4], l[4];
                            #pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (kPlanes == 3)
                                    thirds(v[8 * q + 2 * i], v[8 * q + 2 * i + 1], h[i], m[i], l[i]);
                                else
                                    h[i] = pack(v[8 * q + 2 * i], v[8 * q + 2 * i + 1], E{});
                            }
                            *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                            if (kPlanes == 3) {
                                *reinterpret_cast<uint4*>(to + kPlane) = make_uint4(m[0], m[1], m[2], m[3]);
                                *reinterpret_cast<uint4*>(to + 2 * kPlane) = make_uint4(l[0], l[1], l[2], l[3]);
                            }
                        }
                        if (here) {
                            uint16_t* p = reinterpret_cast<uint16_t*>(out + g_unit<kSpan>(lane, q0 + (int)rel / 8)) + rel % 8;
                            if (kPlanes == 3) {
                                uint32_t h, m, l;
                                thirds(gy, 0.f, h, m, l);
                                p[0] = (uint16_t)h;
                                p[kPlane / 2] = (uint16_t)m;
                                p[kPlane] = (uint16_t)l;
                            } else {
                                p[0] = (uint16_t)pack(gy, 0.f, E{});
                            }
                        }
                        // (past the last class the second block holds what it held: nobody reads there)
                        if (ch % kSpan == kSpan - 1 || cb + 32 >= a.cols) {
                            tc::fence_async_smem();
                            __syncwarp();
                            if (lane == 0 && y0 < a.rows) {
                                tc::store_2d(&a.out[0], out_addr, (int)cb - 8 * q0, (int)y0);
                                if (kPlanes == 3) {
                                    tc::store_2d(&a.out[1], out_addr + kPlane, (int)cb - 8 * q0, (int)y0);
                                    tc::store_2d(&a.out[2], out_addr + 2 * kPlane, (int)cb - 8 * q0, (int)y0);
                                }
                                tc::store_commit();
                            }
                        }
                        if (a.bias_part) {
                            // the bias's gradient from g before its rounding: 32 rows' sums a column
                            float c = column_sums(v, lane);
                            while (hit) {
                                const int l = __ffs(hit) - 1;
                                hit &= hit - 1;
                                const int at = __shfl_sync(0xffffffffu, (int)rel, l);
                                const float wl = __shfl_sync(0xffffffffu, wt, l);
                                if (lane == at) c -= wl;
                            }
                            if (cb + lane < a.ldg) a.bias_part[((int64_t)mt * 4 + quarter) * a.ldg + cb + lane] = c;
                        }
                    } else {
                        // sums of earlier pieces: dx of class pieces, dw of row pieces
                        float* keep = a.sums + t.split * a.split_stride +
                                      ((a.tile0 + (int64_t)mt * a.n_tiles + n) * BN + col) * kBM + quarter * 32 + lane;
                        if (!a.first)
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] += keep[j * kBM];
                        if (!a.last || !a.direct) {
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) keep[j * kBM] = v[j];
                            continue;
                        }
                        using D = typename std::conditional<kPlanes == 3, float, E>::type;
                        const int count = (int)min((int64_t)32, a.cols - cb);
                        if (a.half_g) {
                            const float q = pow2i(-ue);
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= q;
                        }
                        if (MODE == DX && y < 0)
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.f;
                        D* dx = (D*)a.dx + (a.row0 + y0) * a.dxr + cb * a.dxk;
                        if (a.dxr == 1 && a.dxk != 1) {
                            // column by column: neighbouring lanes are neighbouring rows
                            if (valid)
                                #pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (j < count) dx[lane + j * a.dxk] = from_float<D>(v[j]);
                        } else {
                            tc::store_wait_read<0>();
                            out_write<D>(out, lane, v);
                            if (a.dx_map) {
                                tc::fence_async_smem();
                                __syncwarp();
                                if (lane == 0 && y0 < a.rows) {
                                    tc::store_2d(&a.out[0], out_addr, (int)cb, (int)(a.row0 + y0));
                                    tc::store_commit();
                                }
                            } else {
                                // rows that TMA cannot reach: one at a time, a lane a column
                                __syncwarp();
                                const int rows = (int)min((int64_t)32, a.rows - y0);
                                if (lane < count)
                                    #pragma unroll 8
                                    for (int i = 0; i < rows; ++i) dx[i * a.dxr + lane * a.dxk] = *out_at<D>(out, i, lane);
                                __syncwarp();
                            }
                        }
                    }
                }
                if (MODE == LSE) {
                    // columns past the classes hold -inf from their bias (or, a whole block past them, are cut)
                    const int blocks = (int)min((int64_t)(kCols / 32), max((int64_t)0, (a.cols - (int64_t)n * BN - half * kCols + 31) / 32));
                    float m4[4] = {top, top, top, top};
                    #pragma unroll
                    for (int ch = 0; ch < kCols / 32; ++ch)
                        if (ch < blocks)
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], sums[ch * 32 + j]);
                    const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    const float shift = m == -INFINITY ? 0.f : m;   // nothing but excluded classes so far
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
                    #pragma unroll
                    for (int ch = 0; ch < kCols / 32; ++ch)
                        if (ch < blocks)
                            #pragma unroll
                            for (int j = 0; j < 32; ++j) s4[j & 3] += exp_fast(sums[ch * 32 + j] - shift);
                    sum = sum * exp_fast(top - shift) + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
                    top = m;
                }
            }
            if (MODE == LSE && valid) {
                a.part[row * (2 * a.splits) + 2 * t.split + half] = make_float2(top, sum);
                if (!isnan(zy)) a.zy[row] = zy;   // one thread of all has the label's column
            }
        }
        tc::store_wait_all();
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();   // neither CTA leaves while the other's MMAs or arrivals may reach it
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, 2 * BN);
}

// ---- before the products ---------------------------------------------------------------

struct SetupArgs {
    const int64_t* labels;
    int64_t n;
    const float* weight;      // nullable
    int64_t weight_stride;
    float scale;
    int want_weight;          // largest row weight
    const float* bias;
    float* bias_pad;
    int64_t c, c_pad;
    float* zy;                // nullable: cleared to NaN
    uint32_t* keep;           // nullable: bit r of word r / 32: row r counts
    Meta* meta;
};

__global__ void __launch_bounds__(256) xent_setup_kernel(SetupArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t gt = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, all = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = gt; i < a.c_pad; i += all)
        a.bias_pad[i] = i < a.c ? (a.bias ? a.bias[i] : 0.f) : -INFINITY;
    if (!a.want_weight && !a.zy && !a.keep) return;
    float top = 0.f;
    for (int64_t w = gt / 32; w < (a.n + 31) / 32; w += all / 32) {
        const int64_t r = w * 32 + lane;
        const bool in = r < a.n;
        const bool kept = in && a.labels[r] >= 0;
        if (a.zy && in) a.zy[r] = NAN;
        if (a.keep) {
            const uint32_t bits = __ballot_sync(0xffffffffu, kept);
            if (lane == 0) a.keep[w] = bits;
        }
        if (a.want_weight && kept) {
            const float v = fabsf((a.weight ? a.weight[r * a.weight_stride] : 1.f) * a.scale);
            if (v <= 3.402823466e38f) top = fmaxf(top, v);
        }
    }
    if (a.want_weight) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (lane == 0 && m) atomicMax(&a.meta->weight_bits, m);
    }
}

// Looks for left-out rows of a 16-bit x read in place that hold a value that is no number (0 x it
// would be NaN in dw, whose sum runs over the rows); a warp a row.
__global__ void __launch_bounds__(256) xent_poison_kernel(const int64_t* __restrict__ labels, int64_t n,
                                                          const uint16_t* __restrict__ x, int64_t xr, int64_t d, int bf16,
                                                          Meta* meta) {
    const int lane = threadIdx.x & 31;
    const uint32_t inf = bf16 ? 0x7f80 : 0x7c00;
    for (int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32; r < n; r += (int64_t)gridDim.x * blockDim.x / 32) {
        if (labels[r] >= 0) continue;
        bool b = false;
        // rows read in place start on 16 bytes
        const uint4* p = reinterpret_cast<const uint4*>(x + r * xr);
        for (int64_t k = lane; k < d / 8; k += 32) {
            const uint4 q = p[k];
            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
            #pragma unroll
            for (int i = 0; i < 4; ++i) b |= (u[i] & inf) == inf || (u[i] >> 16 & inf) == inf;
        }
        if (lane < d % 8) b |= (x[r * xr + d / 8 * 8 + lane] & inf) == inf;
        if (__any_sync(0xffffffffu, b) && lane == 0) meta->poison = 1;
    }
}

// lse and loss of a row (null: given) from its partial maxima and sums, and the shift of its g
__global__ void __launch_bounds__(256) xent_join_kernel(const float2* __restrict__ part, int parts, int lanes,
                                                        const float* zy, const int64_t* labels, int64_t n,
                                                        float* loss, float* lse, float2* shift, int if_far,
                                                        const Meta* meta) {
    if (if_far && meta->far == 0) return;
    // `lanes` neighbouring threads to a row, 1 or 32
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, r = at / lanes;
    const int lane = (int)(at % lanes);
    if (r >= n) return;
    float m = -INFINITY;
    for (int i = lane; i < parts; i += lanes) m = fmaxf(m, part[r * parts + i].x);
    if (lanes == 32)
        #pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float sh = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int i = lane; i < parts; i += lanes) {
        const float2 p = part[r * parts + i];
        s += p.y * expf(p.x - sh);
    }
    if (lanes == 32)
        #pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane != 0) return;
    const float l = logf(s);
    if (shift) shift[r] = make_float2(sh, l);
    if (!loss) return;
    const bool kept = labels[r] >= 0;
    const bool failed = meta->err != 0;
    loss[r] = failed ? NAN : kept ? (sh - zy[r]) + l : 0.f;
    if (lse) lse[r] = failed ? NAN : kept ? sh + l : 0.f;
}

// The shift that g subtracts where loss and lse are given: lse, as it was rounded.  Past kFarLse its
// last bit (2^-16 and more) shows in every probability of the row, and where a mask has left the
// type's lowest value for all logits, nothing of the log of their sum is left in it.  A call with
// such a row forms the maxima and sums again from the same products (meta->far).
constexpr float kFarLse = 256.f;
__global__ void __launch_bounds__(256) xent_shift_kernel(const int64_t* __restrict__ labels, int64_t n, const float* __restrict__ lse,
                                                         float2* __restrict__ shift, Meta* meta) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= n) return;
    const float l = lse[r];
    shift[r] = make_float2(l, 0.f);
    if (labels[r] >= 0 && fabsf(l) > kFarLse) meta->far = 1;
}

// Rows read four features at a time: unit features, 16-byte aligned rows.
__host__ __device__ inline bool rows_vector(const void* p, int64_t sr, int64_t sk) {
    return sk == 1 && sr >= 0 && (uintptr_t)p % 16 == 0 && sr % 4 == 0;
}
__device__ __forceinline__ float4 load_quad(const float* row, int64_t k, int64_t d) {
    if (k + 4 <= d) return *reinterpret_cast<const float4*>(row + k);
    return make_float4(k < d ? row[k] : 0.f, k + 1 < d ? row[k + 1] : 0.f, k + 2 < d ? row[k + 2] : 0.f, 0.f);
}
__device__ __forceinline__ bool row_counts(const uint32_t* keep, int64_t r) { return (keep[r >> 5] >> (r & 31)) & 1; }

// thirds() of two values; one that is not finite is h alone
__device__ __forceinline__ void split3(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
    thirds(a, b, h, m, l);
    // (a NaN that holds its bits in the lower half would be cut to infinity)
    const bool fa = fabsf(a) <= 3.402823466e38f, fb = fabsf(b) <= 3.402823466e38f;
    if (fa && fb) return;
    h = pack(fa ? __uint_as_float(h << 16) : a, fb ? __uint_as_float(h & 0xffff0000u) : b, __nv_bfloat16{});
    const uint32_t keep = (fa ? 0xffffu : 0u) | (fb ? 0xffff0000u : 0u);
    m &= keep;
    l &= keep;
}

// What the operands' copies are made of and go to: rows x d -> planes [rows][dp], zero past the
// features and in rows with a negative label.
struct PlaneArgs {
    const void* x;
    int64_t xr, xk;
    const uint32_t* keep;     // nullable: bit r of word r / 32: row r counts
    int64_t rows, d, dp;
    int64_t per_block;        // xent_planes_rows_kernel: rows a block
    Meta* meta;
    int if_poison;            // nothing to do unless meta->poison is set
    uint16_t* to[4];          // one plane of 16 bits, or h, m, l of fp32, and (nullable) its infinities
};
// Infinities go from two values to a plane of their own; true when there are any.
__device__ __forceinline__ bool take_infinities(float& a, float& b, uint32_t& plane) {
    const bool ia = isinf(a), ib = isinf(b);
    plane = pack(ia ? a : 0.f, ib ? b : 0.f, __nv_bfloat16{});
    if (ia) a = 0.f;
    if (ib) b = 0.f;
    return ia || ib;
}

// fp32 rows in 16-byte units: a block takes some rows of 1024 features, a thread four of them,
// several rows at once where the features are fewer.
__global__ void __launch_bounds__(256) xent_planes_rows_kernel(const PlaneArgs a) {
    const int64_t blocks_k = (a.dp + 1023) / 1024;
    const int64_t k0 = (blockIdx.x % blocks_k) * 1024, r0 = (blockIdx.x / blocks_k) * a.per_block;
    const int64_t r1 = min(a.rows, r0 + a.per_block);
    const int quads = (int)min((int64_t)256, (a.dp - k0) / 4), at_once = 256 / quads;
    const int quad = threadIdx.x % quads, ro = threadIdx.x / quads;
    if (ro >= at_once) return;
    const int64_t k = k0 + 4 * quad;
    #pragma unroll 4
    for (int64_t r = r0 + ro; r < r1; r += at_once) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!a.keep || row_counts(a.keep, r)) v = load_quad((const float*)a.x + r * a.xr, k, a.d);
        uint2 h, m, l;
        if (a.to[3]) {
            uint2 f;
            const bool some = take_infinities(v.x, v.y, f.x) | take_infinities(v.z, v.w, f.y);
            *reinterpret_cast<uint2*>(a.to[3] + r * a.dp + k) = f;
            if (some) a.meta->wild = 1;
        }
        split3(v.x, v.y, h.x, m.x, l.x);
        split3(v.z, v.w, h.y, m.y, l.y);
        *reinterpret_cast<uint2*>(a.to[0] + r * a.dp + k) = h;
        *reinterpret_cast<uint2*>(a.to[1] + r * a.dp + k) = m;
        *reinterpret_cast<uint2*>(a.to[2] + r * a.dp + k) = l;
    }
}

// any strides, a 64 x 64 tile a block; T: type of x, E: of the planes
template <typename T, typename E>
__global__ void __launch_bounds__(256) xent_planes_kernel(const PlaneArgs a) {
    __shared__ float t[64][65];      // [feature][row]
    if (a.if_poison && a.meta->poison == 0) return;
    const int64_t tiles_k = (a.dp + 63) / 64;
    const int64_t k0 = (blockIdx.x % tiles_k) * 64, r0 = (blockIdx.x / tiles_k) * 64;
    const T* x = (const T*)a.x;
    const bool down = a.xr == 1 && a.xk != 1;
    if (down && sizeof(T) == 4 && (uintptr_t)x % 16 == 0 && a.xk % 4 == 0) {
        // four rows of a feature at a time
        #pragma unroll
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = (i & 15) * 4, k = i >> 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r0 + r < a.rows && k0 + k < a.d) {
                v = load_quad((const float*)x + (k0 + k) * a.xk, r0 + r, a.rows);
                const uint32_t bits = a.keep ? a.keep[(r0 + r) >> 5] >> ((r0 + r) & 31) : 15;
                if (!(bits & 1)) v.x = 0.f;
                if (!(bits & 2)) v.y = 0.f;
                if (!(bits & 4)) v.z = 0.f;
                if (!(bits & 8)) v.w = 0.f;
            }
            t[k][r] = v.x;
            t[k][r + 1] = v.y;
            t[k][r + 2] = v.z;
            t[k][r + 3] = v.w;
        }
    } else {
        #pragma unroll 8
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = down ? i & 63 : i >> 6, k = down ? i >> 6 : i & 63;
            float v = 0.f;
            if (r0 + r < a.rows && k0 + k < a.d && (!a.keep || row_counts(a.keep, r0 + r)))
                v = to_float(x[(r0 + r) * a.xr + (k0 + k) * a.xk]);
            t[k][r] = v;
        }
    }
    __syncthreads();
    // 8 features of a row to a thread, 16 bytes of a plane
    const int k = (threadIdx.x & 7) * 8;
    if (k0 + k >= a.dp) return;
    #pragma unroll
    for (int r = threadIdx.x >> 3; r < 64; r += 32) {
        if (r0 + r >= a.rows) break;
        const int64_t at = (r0 + r) * a.dp + k0 + k;
        uint32_t h[4], m[4], l[4], f[4];
        bool some = false;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v0 = t[k + 2 * i][r], v1 = t[k + 2 * i + 1][r];
            if constexpr (sizeof(T) == 4) {
                if (a.to[3]) some |= take_infinities(v0, v1, f[i]);
                split3(v0, v1, h[i], m[i], l[i]);
            } else {
                h[i] = pack(v0, v1, E{});
            }
        }
        if constexpr (sizeof(T) == 4)
            if (a.to[3]) {
                *reinterpret_cast<uint4*>(a.to[3] + at) = make_uint4(f[0], f[1], f[2], f[3]);
                if (some) a.meta->wild = 1;
            }
        *reinterpret_cast<uint4*>(a.to[0] + at) = make_uint4(h[0], h[1], h[2], h[3]);
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint4*>(a.to[1] + at) = make_uint4(m[0], m[1], m[2], m[3]);
            *reinterpret_cast<uint4*>(a.to[2] + at) = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
}

// ---- after the products ----------------------------------------------------------------

// the bias's gradient from sums of 32 rows: 32 columns a block, one split of the lines
__global__ void __launch_bounds__(256) xent_colsum_kernel(const float* __restrict__ sums, int64_t ldg, int64_t lines,
                                                          int64_t cols, int64_t per_split, int first,
                                                          double* __restrict__ part, int64_t c_total, int64_t c0) {
    __shared__ double s[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + tx;
    const int64_t r0 = blockIdx.y * per_split, r1 = min(lines, r0 + per_split);
    double v = 0.0;
    if (col < cols) {
        #pragma unroll 4
        for (int64_t r = r0 + ty; r < r1; r += 8) v += (double)sums[r * ldg + col];
    }
    s[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && col < cols) {
        v = 0.0;
        for (int i = 0; i < 8; ++i) v += s[i][tx];
        double* p = part + blockIdx.y * c_total + c0 + col;
        *p = first ? v : *p + v;
    }
}

// The end of a gradient call: dbias from its splits; and, where a kernel's wait gave up, NaN in
// everything that the call writes (loss and lse null: given).
template <typename T>
struct FinishArgs {
    const Meta* meta;
    int half_g, bias_splits;
    int64_t n, d, c;
    T *dx, *dw;
    int64_t dxr, dxk;
    const double* bias_part;
    float *dbias, *loss, *lse;
};
template <typename T>
__global__ void __launch_bounds__(256) xent_finish_kernel(const FinishArgs<T> a) {
    const bool failed = a.meta->err != 0;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    if (a.dbias)
        for (int64_t j = at / 32; j < a.c; j += all / 32) {   // a warp a class
            double v = 0.0;
            for (int s = threadIdx.x & 31; s < a.bias_splits; s += 32) v += a.bias_part[s * a.c + j];
            #pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if ((threadIdx.x & 31) == 0) a.dbias[j] = failed ? NAN : (float)ldexp(v, -g_exponent(a.meta, a.half_g));
        }
    if (!failed) return;
    if (a.dw)
        for (int64_t i = at; i < a.c * a.d; i += all) a.dw[i] = from_float<T>(NAN);
    if (a.dx)
        for (int64_t i = at; i < a.n * a.d; i += all) a.dx[i / a.d * a.dxr + i % a.d * a.dxk] = from_float<T>(NAN);
    if (a.loss)
        for (int64_t i = at; i < a.n; i += all) a.loss[i] = NAN;
    if (a.lse)
        for (int64_t i = at; i < a.n; i += all) a.lse[i] = NAN;
}

// dw or dx from several splits' sums: a block makes 32 rows x 8 features, a warp a feature.  Rows
// with a negative label (dx) are zero.
template <typename T>
__global__ void __launch_bounds__(256) xent_sum_kernel(const float* __restrict__ sums, int splits, int64_t split_stride,
                                                       int n_tiles, int bn, int64_t rows, int d, int half_g,
                                                       const Meta* __restrict__ meta, const int64_t* __restrict__ labels,
                                                       T* __restrict__ out, int64_t out_row, int64_t out_col) {
    __shared__ float t[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int tiles_k = (d + 7) / 8;
    const int k0 = (int)(blockIdx.x % tiles_k) * 8, k = k0 + ty;
    const int64_t r0 = (int64_t)(blockIdx.x / tiles_k) * 32;
    if (k < d && r0 + tx < rows) {
        const float* p = sums + ((r0 / kBM * n_tiles + k / bn) * bn + k % bn) * kBM + r0 % kBM + tx;
        double v = 0.0;
        #pragma unroll 8
        for (int s = 0; s < splits; ++s) v += (double)p[s * split_stride];
        float f = scale2((float)v, -g_exponent(meta, half_g));
        if (labels && labels[r0 + tx] < 0) f = 0.f;
        t[ty][tx] = f;
    }
    __syncthreads();
    // neighbouring threads on neighbouring elements of the output
    const bool down = out_row == 1;
    const int j = down ? tx : threadIdx.x >> 3, i = down ? ty : threadIdx.x & 7;
    if (r0 + j < rows && k0 + i < d) out[(r0 + j) * out_row + (k0 + i) * out_col] = from_float<T>(t[i][j]);
}

// ---- host ------------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    return fn;
}

// rows of `inner` values, `ld` apart, written in blocks of 32 rows x `cols`
bool make_out_map(CUtensorMap* map, int type, const void* base, int64_t inner, int64_t rows, int64_t ld, int cols = 32) {
    auto enc = encoder();
    if (!enc) return false;
    const bool wide = type == GAFIME_TYPE_FP32;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * (wide ? 4 : 2)};
    cuuint32_t box[2] = {(cuuint32_t)cols, 32};
    cuuint32_t estr[2] = {1, 1};
    return enc(map,
               wide                          ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
               : type == GAFIME_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
               2, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               cols * (wide ? 4 : 2) == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows of `inner` 16-bit values, `ld` apart; boxes of 64 values x box_rows
bool make_map(CUtensorMap* map, bool bf16, const void* base, int64_t inner, int64_t rows, int64_t ld, int box_rows) {
    auto enc = encoder();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)base, dims,
               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// columns of an accumulator tile: the smallest that holds the axis, 256 past that
int tile_n(int64_t cols) { return cols <= 64 ? 64 : cols <= 128 ? 128 : 256; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// TMA reads 16-bit rows in place: contiguous rows, 16-byte aligned base and pitch
bool in_place(int type, const void* p, int64_t row, int64_t col, int64_t len) {
    return type != GAFIME_TYPE_FP32 && col == 1 && row >= len && (uintptr_t)p % 16 == 0 && row % 8 == 0;
}

struct Plan {
    int planes, bn_c, bn_dx, bn_dw;
    bool x_in_place, w_in_place;
    int64_t dp;
    int64_t m_tiles, c_tiles;        // of the whole call, 256 rows and bn_c classes
    int splits, per_split;           // LSE
    int64_t piece_rows, piece_classes, ldg;
    int64_t dx_d_tiles;              // of bn_dx features
    int64_t dx_stride;               // floats of a split's sums
    int dx_splits, dx_per_split;
    bool dx_direct;                  // one split: dx leaves the products' kernel
    int64_t dw_c_tiles, dw_d_tiles;  // 128 classes x bn_dw features
    int64_t dw_stride;               // floats of a split's partial
    int dw_splits, dw_per_split;
    bool dw_direct;                  // one split: dw leaves the products' kernel
    int bias_splits;
    bool products;                   // dx or dw or dbias wanted
    // workspace
    Meta* meta;
    float* bias;
    uint32_t* keep;
    uint16_t* xc;                    // x without left-out rows, made where one of those holds no number
    uint16_t *x[3], *w[4], *g[3];    // planes; null where the operands are read in place
    float2* part;
    float* zy;
    float2* shift;
    float* dx_sums;
    float* dw_part;
    float* bias_sums;
    double* bias_part;
    size_t bytes;
};

Plan make_plan(const XentCall& a, int sms, uint8_t* ws) {
    Plan p{};
    p.planes = a.type == GAFIME_TYPE_FP32 ? 3 : 1;
    p.bn_c = tile_n(a.c);
    const int pairs = sms / 2;
    p.x_in_place = in_place(a.type, a.x, a.xr, a.xk, a.d);
    p.w_in_place = in_place(a.type, a.w, a.wr, a.wk, a.d);
    p.dp = up(a.d, 8);
    p.m_tiles = std::max<int64_t>(1, cdiv(a.n, kPM));
    p.c_tiles = cdiv(a.c, p.bn_c);
    // LSE: units of (row tile, run of class tiles), the longest runs that leave the pairs of CTAs
    // about as evenly loaded as any
    auto load = [&](int64_t run) { return cdiv(p.m_tiles * cdiv(p.c_tiles, run), pairs) * run; };
    int64_t best = load(p.c_tiles);
    for (int64_t run = 1; run < p.c_tiles && run <= 64; ++run) best = std::min(best, load(run));
    int64_t run = p.c_tiles;
    if (load(run) > best + best / 32)
        for (run = std::min<int64_t>(64, p.c_tiles); run > 1 && load(run) > best + best / 32;) --run;
    p.per_split = (int)run;
    p.splits = (int)cdiv(p.c_tiles, p.per_split);
    p.products = a.gradient && (a.dx || a.dw || a.dbias) && a.n > 0;

    Carver cv(ws);
    p.meta = cv.take<Meta>(1);
    p.bias = cv.take<float>(p.c_tiles * p.bn_c + 256);
    p.keep = cv.take<uint32_t>(cdiv(a.n, 32) + 2);
    for (int i = 0; i < p.planes; ++i) {
        if (!p.x_in_place) p.x[i] = cv.take<uint16_t>(std::max<int64_t>(1, a.n) * p.dp);
        if (!p.w_in_place) p.w[i] = cv.take<uint16_t>(a.c * p.dp);
    }
    if (p.planes == 3) p.w[3] = cv.take<uint16_t>(a.c * p.dp);
    if (a.gradient && a.dw && p.x_in_place) p.xc = cv.take<uint16_t>(std::max<int64_t>(1, a.n) * p.dp);
    p.part = cv.take<float2>(a.n * 2 * p.splits);
    p.zy = cv.take<float>(a.n);
    if (p.products) {
        p.shift = cv.take<float2>(a.n);
        // a piece of g: rows for one row tile an SM, then as many classes as piece_bytes hold
        const int64_t es = 2 * p.planes;
        p.piece_rows = std::min<int64_t>(up(a.n, kPM), (int64_t)pairs * kPM);
        p.piece_classes = std::max<int64_t>(1024, (int64_t)(piece_bytes(p.planes) / (p.piece_rows * es)) / 256 * 256);
        if (p.piece_classes >= a.c) {
            p.piece_classes = a.c;
            // few classes: more rows at once, still whole rounds of the SMs
            const int64_t more = (int64_t)(piece_bytes(p.planes) / (p.piece_rows * es * up(a.c, 8)));
            if (more > 1) p.piece_rows = std::min<int64_t>(up(a.n, kPM), p.piece_rows * more);
        }
        p.ldg = up(p.piece_classes, 64);   // whole 128-byte lines: TMA boxes meet no line twice
        for (int i = 0; i < p.planes; ++i) p.g[i] = cv.take<uint16_t>(p.piece_rows * p.ldg);
        // Feature tiles of 128 or 256 (a CTA's half is whole 64-value lines), and the sum over classes
        // (dx) or rows (dw) split over pairs that the tiles leave idle, in runs of at least 4 blocks:
        // what takes the fewest rounds, where a block of 128 takes about 0.6 of one of 256
        auto choose = [&](int64_t row_tiles, int64_t blocks, int& bn_out, int& per_out) {
            double best = 1e300;
            for (int bn : {256, 128}) {
                if (bn == 256 && a.d <= 128) continue;
                const int64_t tiles = row_tiles * cdiv(a.d, bn);
                for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(pairs, blocks / 4)); ++s) {
                    const int64_t per = cdiv(blocks, s);
                    if (s > 1 && tiles * cdiv(blocks, per) > 2 * pairs) break;
                    const double cost = cdiv(tiles * cdiv(blocks, per), pairs) * (per + 4.0) * (bn == 256 ? 1.0 : 0.6);
                    if (cost < best * 0.97) {
                        best = cost;
                        bn_out = bn;
                        per_out = (int)per;
                    }
                }
            }
        };
        const int64_t rows_at_once = std::min(a.n, p.piece_rows), blocks = cdiv(rows_at_once, kBK);
        const int64_t class_blocks = cdiv(p.piece_classes, kBK);
        choose(cdiv(rows_at_once, kPM), class_blocks, p.bn_dx, p.dx_per_split);
        choose(cdiv(p.piece_classes, kPM), blocks, p.bn_dw, p.dw_per_split);
        p.dx_splits = (int)cdiv(class_blocks, p.dx_per_split);
        p.dx_direct = p.dx_splits == 1;
        p.dw_splits = (int)cdiv(blocks, p.dw_per_split);
        p.dx_d_tiles = cdiv(a.d, p.bn_dx);
        p.dw_d_tiles = cdiv(a.d, p.bn_dw);
        p.dx_stride = p.piece_rows * p.dx_d_tiles * p.bn_dx;
        p.dw_c_tiles = cdiv(a.c, kPM) * 2;
        p.dw_stride = p.dw_c_tiles * p.dw_d_tiles * p.bn_dw * kBM;
        if (a.dx && (!p.dx_direct || p.piece_classes < a.c)) p.dx_sums = cv.take<float>(p.dx_splits * p.dx_stride);
        if (a.dw) {
            p.dw_direct = p.dw_splits == 1;
            if (!p.dw_direct || a.n > p.piece_rows) p.dw_part = cv.take<float>(p.dw_splits * p.dw_stride);
        }
        if (a.dbias) {
            const int64_t blocks = cdiv(p.piece_classes, 32);
            p.bias_splits = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(4 * sms, blocks), cdiv(p.piece_rows, 32 * 16)));
            p.bias_sums = cv.take<float>(p.piece_rows / 32 * p.ldg);
            p.bias_part = cv.take<double>(p.bias_splits * a.c);
        }
    }
    p.bytes = cv.used;
    return p;
}

template <int MODE, int BN, typename E, int kPlanes>
cudaError_t launch_bn(const TcArgs& t, int sms, cudaStream_t stream) {
    auto fn = xent_tc_kernel<MODE, BN, E, kPlanes>;
    static std::atomic<uint64_t> ready{0};   // devices on which the kernel has its shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !((ready.load(std::memory_order_relaxed) >> dev) & 1)) {
        e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(BN, out_bytes(MODE, kPlanes)));
        if (e != cudaSuccess) return e;
        // the epilogues take their registers from the launch's: one that has fewer would wait for good
        cudaFuncAttributes attr;
        e = cudaFuncGetAttributes(&attr, (const void*)fn);
        if (e != cudaSuccess) return e;
        if (attr.numRegs * kThreads < 128 * kControlRegs + 256 * kEpiRegs) return cudaErrorLaunchOutOfResources;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    KernelTimer kt(stream, GAFIME_KERNEL_XENT_TC);
    fn<<<2 * std::min(sms / 2, t.units), kThreads, smem_of(BN, out_bytes(MODE, kPlanes)), stream>>>(t);
    return cudaGetLastError();
}
template <int MODE, typename E, int kPlanes>
cudaError_t launch(const TcArgs& t, int bn, int sms, cudaStream_t stream) {
    if (t.units <= 0) return cudaSuccess;
    switch (bn) {
        case 64: return launch_bn<MODE, 64, E, kPlanes>(t, sms, stream);
        case 128: return launch_bn<MODE, 128, E, kPlanes>(t, sms, stream);
        default: return launch_bn<MODE, 256, E, kPlanes>(t, sms, stream);
    }
}

#define XENT_TRY(expr)                                \
    do {                                              \
        const cudaError_t e_ = (expr);                \
        if (e_ != cudaSuccess) return e_;             \
    } while (0)

template <typename T, typename E>
cudaError_t planes(PlaneArgs s, int sms, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        if (rows_vector(s.x, s.xr, s.xk)) {
            const int64_t blocks_k = cdiv(s.dp, 1024);
            s.per_block = std::max<int64_t>(16, cdiv(s.rows * blocks_k, 16 * sms));
            KernelTimer kt(stream, GAFIME_KERNEL_XENT);
            xent_planes_rows_kernel<<<(unsigned)(blocks_k * cdiv(s.rows, s.per_block)), 256, 0, stream>>>(s);
            return cudaGetLastError();
        }
    }
    KernelTimer kt(stream, GAFIME_KERNEL_XENT);
    xent_planes_kernel<T, E><<<(unsigned)(cdiv(s.dp, 64) * cdiv(s.rows, 64)), 256, 0, stream>>>(s);
    return cudaGetLastError();
}

std::atomic<int> fail_waits{0};   // gafime_xent_fail_waits

template <typename T, typename E>
cudaError_t run_tc(const XentCall& a, int sms) {
    const Plan p = make_plan(a, sms, a.ws);
    constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
    constexpr int kPlanes = std::is_same<T, float>::value ? 3 : 1;
    cudaStream_t st = a.stream;
    if (a.n == 0) {   // gradients of no rows
        if (a.dw) XENT_TRY(cudaMemsetAsync(a.dw, 0, (size_t)(a.c * a.d) * sizeof(T), st));
        if (a.dbias) XENT_TRY(cudaMemsetAsync(a.dbias, 0, a.c * 4, st));
        return cudaSuccess;
    }
    XENT_TRY(cudaMemsetAsync(p.meta, 0, sizeof(Meta), st));
    if (fail_waits.load(std::memory_order_relaxed)) XENT_TRY(cudaMemsetAsync(&p.meta->err, 1, sizeof(int), st));
    // one tile of classes: the call's losses come with its g, which its own sums normalise
    const bool both = p.products && p.c_tiles == 1;
    const bool forward = !a.have_lse && !both, again = a.have_lse && p.products && !both;
    {
        SetupArgs s{};
        s.labels = a.labels; s.n = a.n; s.weight = a.weight; s.weight_stride = a.weight_stride; s.scale = a.scale;
        s.want_weight = p.products && !kBf16;
        s.bias = a.bias; s.bias_pad = p.bias; s.c = a.c; s.c_pad = p.c_tiles * p.bn_c + 256;
        s.zy = forward || again ? p.zy : nullptr;
        s.keep = p.x[0] || p.xc ? p.keep : nullptr;
        s.meta = p.meta;
        const int64_t threads = std::max<int64_t>(s.c_pad, a.n);
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        xent_setup_kernel<<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(8 * sms, cdiv(threads, 256))), 256, 0, st>>>(s);
        XENT_TRY(cudaGetLastError());
    }
    if (p.xc) {
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        xent_poison_kernel<<<(unsigned)std::min<int64_t>(8 * sms, cdiv(a.n, 8)), 256, 0, st>>>(
            a.labels, a.n, (const uint16_t*)a.x, a.xr, a.d, kBf16, p.meta);
        XENT_TRY(cudaGetLastError());
        PlaneArgs s{a.x, a.xr, a.xk, p.keep, a.n, a.d, p.dp, 0, p.meta, 1, {p.xc}};
        XENT_TRY((planes<T, E>(s, sms, st)));
    }
    if (p.x[0]) {
        PlaneArgs s{a.x, a.xr, a.xk, p.keep, a.n, a.d, p.dp, 0, p.meta, 0, {p.x[0], p.x[1], p.x[2]}};
        XENT_TRY((planes<T, E>(s, sms, st)));
    }
    if (p.w[0]) {
        PlaneArgs s{a.w, a.wr, a.wk, nullptr, a.c, a.d, p.dp, 0, p.meta, 0, {p.w[0], p.w[1], p.w[2], p.w[3]}};
        XENT_TRY((planes<T, E>(s, sms, st)));
    }
    // where the operands are read
    const void *xs[3] = {p.x[0] ? (const void*)p.x[0] : a.x, p.x[1], p.x[2]};
    const void *ws[4] = {p.w[0] ? (const void*)p.w[0] : a.w, p.w[1], p.w[2], p.w[3]};
    const int64_t ldx = p.x[0] ? p.dp : a.xr, ldw = p.w[0] ? p.dp : a.wr;
    auto map = [&](auto& m, const auto& base, int64_t inner, int64_t rows, int64_t ld, int box) {
        for (size_t i = 0; i < std::size(base) && base[i]; ++i)
            if (!make_map(&m[i], kBf16, base[i], inner, rows, ld, box)) return cudaErrorInvalidValue;
        return cudaSuccess;
    };

    TcArgs t{};
    // k blocks summed in tensor memory at a time.  fp32: one, 4 products of the h planes, each cutting
    // about 2^-24 of the sum.  16 bits: 32 products and more are nothing beside the operands' rounding.
    t.chunk = p.planes == 3 ? 1 : 8;
    t.half_g = !kBf16;
    t.meta = p.meta;
    t.bias = p.bias;
    t.labels = a.labels;
    t.weight = a.weight; t.weight_stride = a.weight_stride; t.scale = a.scale;
    t.c_total = a.c;
    t.splits = p.splits;
    if (again) {
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        xent_shift_kernel<<<(unsigned)cdiv(a.n, 256), 256, 0, st>>>(a.labels, a.n, a.lse, p.shift, p.meta);
        XENT_TRY(cudaGetLastError());
    }
    if (forward || again) {
        TcArgs l = t;
        l.if_far = again;
        XENT_TRY(map(l.a, xs, a.d, a.n, ldx, kBM));
        XENT_TRY(map(l.b, ws, a.d, a.c, ldw, p.bn_c / 2));
        l.m_tiles = (int)p.m_tiles;
        l.n_tiles = (int)p.c_tiles;
        l.per_split = p.per_split;
        l.units = l.m_tiles * p.splits;
        l.k_blocks = (int)cdiv(a.d, kBK);
        l.rows = a.n;
        l.cols = a.c;
        l.part = p.part;
        l.zy = p.zy;
        XENT_TRY((launch<LSE, E, kPlanes>(l, p.bn_c, sms, st)));
    }
    if (forward || again) {
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        const int lanes = p.splits >= 16 ? 32 : 1;
        xent_join_kernel<<<(unsigned)cdiv(a.n * lanes, 256), 256, 0, st>>>(
            p.part, 2 * p.splits, lanes, p.zy, a.labels, a.n, forward ? a.loss : nullptr, forward ? a.lse : nullptr,
            p.products ? p.shift : nullptr, again, p.meta);
        XENT_TRY(cudaGetLastError());
    }
    if (!p.products) return cudaSuccess;

    const void* gs[3] = {p.g[0], p.g[1], p.g[2]};
    for (int64_t r0 = 0; r0 < a.n; r0 += p.piece_rows) {
        const int64_t rows = std::min(p.piece_rows, a.n - r0);
        for (int64_t c0 = 0; c0 < a.c; c0 += p.piece_classes) {
            const int64_t classes = std::min(p.piece_classes, a.c - c0);
            TcArgs g = t;
            XENT_TRY(map(g.a, xs, a.d, a.n, ldx, kBM));
            XENT_TRY(map(g.b, ws, a.d, a.c, ldw, p.bn_c / 2));
            g.m_tiles = (int)cdiv(rows, kPM);
            g.n_tiles = (int)cdiv(classes, p.bn_c);
            g.units = g.m_tiles * g.n_tiles;
            g.k_blocks = (int)cdiv(a.d, kBK);
            g.a_row0 = (int)r0;
            g.b_row0 = (int)c0;
            g.rows = rows;
            g.row0 = r0;
            g.cols = classes;
            g.c0 = (int)c0;
            g.shift = p.shift;
            g.loss = a.loss;
            for (int i = 0; i < p.planes; ++i)
                if (!make_out_map(&g.out[i], kBf16 ? GAFIME_TYPE_BF16 : GAFIME_TYPE_FP16, gs[i], p.ldg, rows, p.ldg,
                                  p.bn_c >= 128 ? 64 : 32))
                    return cudaErrorInvalidValue;
            g.ldg = p.ldg;
            g.bias_part = a.dbias ? p.bias_sums : nullptr;
            g.loss_out = a.have_lse ? nullptr : a.loss;
            g.lse_out = a.lse;
            if (both)
                XENT_TRY((launch<BOTH, E, kPlanes>(g, p.bn_c, sms, st)));
            else
                XENT_TRY((launch<G, E, kPlanes>(g, p.bn_c, sms, st)));
            if (a.dbias) {
                const int64_t lines = g.m_tiles * 8;
                KernelTimer kt(st, GAFIME_KERNEL_XENT);
                xent_colsum_kernel<<<dim3((unsigned)cdiv(classes, 32), (unsigned)p.bias_splits), 256, 0, st>>>(
                    p.bias_sums, p.ldg, lines, classes, cdiv(p.piece_rows / 32, p.bias_splits), r0 == 0, p.bias_part,
                    a.c, c0);
                XENT_TRY(cudaGetLastError());
            }
            if (a.dx) {
                TcArgs x = t;
                XENT_TRY(map(x.a, gs, classes, rows, p.ldg, kBM));
                // the piece's classes of w
                const void* wp[4] = {};
                for (int i = 0; i < 4 && ws[i]; ++i) wp[i] = (const uint16_t*)ws[i] + c0 * ldw;
                XENT_TRY(map(x.b, wp, a.d, classes, ldw, kBK));
                x.m_tiles = (int)cdiv(rows, kPM);
                x.n_tiles = (int)p.dx_d_tiles;
                x.units = x.m_tiles * x.n_tiles * p.dx_splits;
                x.per_split = p.dx_per_split;
                x.k_blocks = (int)cdiv(classes, kBK);
                if (p.planes == 1) x.chunk = 16;
                x.rows = rows;
                x.row0 = r0;
                x.cols = a.d;
                x.dx = a.dx; x.dxr = a.dxr; x.dxk = a.dxk;
                x.dx_map = a.dxk == 1 && (uintptr_t)a.dx % 16 == 0 && a.dxr >= a.d && a.dxr * (int64_t)sizeof(T) % 16 == 0;
                if (x.dx_map && !make_out_map(&x.out[0], a.type, a.dx, a.d, a.n, a.dxr)) return cudaErrorInvalidValue;
                x.sums = p.dx_sums;
                x.split_stride = p.dx_stride;
                x.direct = p.dx_direct;
                x.first = c0 == 0;
                x.last = c0 + classes == a.c;
                XENT_TRY((launch<DX, E, kPlanes>(x, p.bn_dx, sms, st)));
                if (x.last && !p.dx_direct) {
                    KernelTimer kt(st, GAFIME_KERNEL_XENT);
                    xent_sum_kernel<T><<<(unsigned)(cdiv(rows, 32) * cdiv(a.d, 8)), 256, 0, st>>>(
                        p.dx_sums, p.dx_splits, p.dx_stride, (int)p.dx_d_tiles, p.bn_dx, rows, (int)a.d,
                        !kBf16, p.meta, a.labels + r0, (T*)a.dx + r0 * a.dxr, a.dxr, a.dxk);
                    XENT_TRY(cudaGetLastError());
                }
            }
            if (a.dw) {
                TcArgs w = t;
                XENT_TRY(map(w.a, gs, classes, rows, p.ldg, kBK));
                XENT_TRY(map(w.b, xs, a.d, a.n, ldx, kBK));
                w.m_tiles = (int)cdiv(classes, kPM);
                w.n_tiles = (int)p.dw_d_tiles;
                w.units = w.m_tiles * w.n_tiles * p.dw_splits;
                w.per_split = p.dw_per_split;
                w.k_blocks = (int)cdiv(rows, kBK);
                if (p.planes == 1) w.chunk = 16;
                w.b_row0 = (int)r0;
                w.row0 = c0;
                w.rows = classes;
                w.cols = a.d;
                w.first = r0 == 0;
                w.last = r0 + rows == a.n;
                w.sums = p.dw_part;
                w.split_stride = p.dw_stride;
                w.tile0 = c0 / kBM * p.dw_d_tiles;
                w.direct = p.dw_direct;
                w.dx = a.dw;
                w.dxr = a.d;
                w.dxk = 1;
                w.dx_map = (uintptr_t)a.dw % 16 == 0 && a.d * (int64_t)sizeof(T) % 16 == 0;
                if (w.dx_map && !make_out_map(&w.out[0], a.type, a.dw, a.d, a.c, a.d)) return cudaErrorInvalidValue;
                w.cleaned = p.xc != nullptr;
                if (p.xc && !make_map(&w.b[1], kBf16, p.xc, a.d, a.n, p.dp, kBK)) return cudaErrorInvalidValue;
                XENT_TRY((launch<DW, E, kPlanes>(w, p.bn_dw, sms, st)));
            }
        }
    }
    if (a.dw && !p.dw_direct) {
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        xent_sum_kernel<T><<<(unsigned)(cdiv(a.c, 32) * cdiv(a.d, 8)), 256, 0, st>>>(
            p.dw_part, p.dw_splits, p.dw_stride, (int)p.dw_d_tiles, p.bn_dw, a.c, (int)a.d, !kBf16, p.meta, nullptr, (T*)a.dw, a.d, 1);
        XENT_TRY(cudaGetLastError());
    }
    {
        FinishArgs<T> f{};
        f.meta = p.meta; f.half_g = !kBf16; f.bias_splits = p.bias_splits;
        f.n = a.n; f.d = a.d; f.c = a.c;
        f.dx = (T*)a.dx; f.dxr = a.dxr; f.dxk = a.dxk;
        f.dw = (T*)a.dw;
        f.bias_part = p.bias_part; f.dbias = a.dbias;
        if (!a.have_lse) f.loss = a.loss, f.lse = a.lse;
        KernelTimer kt(st, GAFIME_KERNEL_XENT);
        xent_finish_kernel<T><<<(unsigned)std::min<int64_t>(2 * sms, cdiv(a.c, 8)), 256, 0, st>>>(f);
        XENT_TRY(cudaGetLastError());
    }
    return cudaSuccess;
}

}  // namespace

size_t xent_tc_workspace(const XentCall& a, int sms) { return make_plan(a, sms, nullptr).bytes; }

cudaError_t xent_tc(const XentCall& a, int sms) {
    switch (a.type) {
        case GAFIME_TYPE_FP32: return run_tc<float, __nv_bfloat16>(a, sms);
        case GAFIME_TYPE_FP16: return run_tc<__half, __half>(a, sms);
        default: return run_tc<__nv_bfloat16, __nv_bfloat16>(a, sms);
    }
}

}  // namespace gafime

extern "C" int gafime_xent_fail_waits(int enable) {
    gafime::fail_waits.store(enable != 0);
    return GAFIME_SUCCESS;
}
