// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + scale[a] (x[t] A[a]) B[a],   a = the adapter of token t's session (or none).
//
// Three kernels.  `plan` sorts the tokens by adapter on the device, once per batch: a stable order
// (adapter, then token) and a list of tiles of up to 64 rows of one adapter, so that the products
// share an adapter's weights between its sessions.  `shrink` computes h = x A per (tile, slice of the
// inputs) into fp32 partials; `expand` sums a tile's partials in slice order, rounds scale * h once to
// bf16 (the operand type; an error of at most 2^-8 of the adapter's own contribution) and adds h B
// to y in fp32, rounded once.  No atomics: the same bits in every run.  In most decode
// batches `few` does the work of both in one launch.
//
// Both products have a rank of 16 to 128 on one side, so the work is bound by moving x, y, A and B:
// tiles come in by cp.async several stages ahead (rows of x and y are gathered, 16 bytes a copy),
// the products are warp-level m16n8k16.
#include "lf_common.cuh"
#include "pool_common.cuh"
#include "sm100_primitives.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace lf {
namespace lora {

namespace cg = cooperative_groups;

constexpr int kTile = 64;                              // rows of a tile
constexpr int kMaxAdapters = 4096;
constexpr int kHeader = 4;                             // ints before the tiles: [0] = number of tiles

// Layout of a plan (int32): header, tiles [max_tiles][4] = {adapter (-1: none), first row, rows, 0},
// order [total] = token of every sorted row, starts [n] = first sorted row of every session.
struct Plan {
    int32_t *head, *tiles, *order, *starts;
};
inline long max_tiles(int total, int n, int adapters) {
    const long parts = n < adapters + 1 ? n : adapters + 1;
    return (total + kTile - 1) / kTile + parts;
}
inline Plan views(int32_t* p, int total, int n, int adapters) {
    Plan v;
    v.head = p;
    v.tiles = p + kHeader;
    v.order = v.tiles + 4 * max_tiles(total, n, adapters);
    v.starts = v.order + total;
    return v;
}

// One CTA.  Bucket b < adapters holds adapter b's sessions, bucket `adapters` those without one.
__global__ void __launch_bounds__(pool::kMetaThreads)
plan_kernel(const int32_t* ids, const int32_t* cu, int n, int total, int adapters,
            Plan p) {
    extern __shared__ int sm[];
    __shared__ int2 buf[32];
    __shared__ int s_big;
    int* tot = sm;                                     // [adapters + 1] tokens
    int* off = sm + adapters + 1;                      // first sorted row
    int* til = off + adapters + 1;                     // first tile
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_wait();
    auto bucket = [&](int i) {
        const int a = ids[i];
        return a >= 0 && a < adapters ? a : adapters;
    };
    // tokens outside [0, total) are cut off: a plan never names a row that does not exist
    auto lo = [&](int i) { return min(max(cu[i], 0), total); };
    auto count = [&](int i) { return max(0, min(max(cu[i + 1], 0), total) - lo(i)); };
    constexpr int kBig = 1024;                         // tokens of a session that the whole CTA copies
    for (int b = threadIdx.x; b <= adapters; b += pool::kMetaThreads) tot[b] = 0;
    if (threadIdx.x == 0) s_big = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += pool::kMetaThreads) {
        const int c = count(i);
        if (c >= kBig) s_big = 1;
        if (c > 0) atomicAdd(&tot[bucket(i)], c);
        if (ids[i] < -1 || ids[i] >= adapters) atomicCAS(&g_device_error, 0, 241);
    }
    __syncthreads();
    int rows = 0, tiles = 0;                           // exclusive sums over the buckets
    for (int b0 = 0; b0 <= adapters; b0 += pool::kMetaThreads) {
        const int b = b0 + threadIdx.x;
        const int c = b <= adapters ? tot[b] : 0, k = (c + kTile - 1) / kTile;
        int xc = c, xk = k;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int oc = __shfl_up_sync(0xffffffffu, xc, d), ok = __shfl_up_sync(0xffffffffu, xk, d);
            if (lane >= d) { xc += oc; xk += ok; }
        }
        if (lane == 31) buf[warp] = make_int2(xc, xk);
        __syncthreads();
        int2 w = buf[lane];                            // every warp scans the warps' sums
        const int2 mine = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int oc = __shfl_up_sync(0xffffffffu, w.x, d), ok = __shfl_up_sync(0xffffffffu, w.y, d);
            if (lane >= d) { w.x += oc; w.y += ok; }
        }
        const int bc = __shfl_sync(0xffffffffu, w.x - mine.x, warp), bk = __shfl_sync(0xffffffffu, w.y - mine.y, warp);
        if (b <= adapters) {
            off[b] = rows + bc + xc - c;
            til[b] = tiles + bk + xk - k;
        }
        rows += __shfl_sync(0xffffffffu, w.x, 31);
        tiles += __shfl_sync(0xffffffffu, w.y, 31);
        __syncthreads();
    }
    // offsets that overlap or leave tokens out give no plan: rows would be written twice or not at all
    if (rows != total || (n > 0 && (cu[0] != 0 || cu[n] != total))) {
        if (threadIdx.x == 0) {
            atomicCAS(&g_device_error, 0, 242);
            p.head[0] = 0;
        }
        return;
    }
    if (threadIdx.x == 0) p.head[0] = tiles;
    __syncthreads();
    for (int b = warp; b <= adapters; b += pool::kMetaThreads / 32) {
        if (tot[b] == 0) continue;
        int run = off[b];
        for (int i0 = 0; i0 < n; i0 += 32) {           // the bucket's sessions, in order
            const int i = i0 + lane;
            const int c = i < n && bucket(i) == b ? count(i) : 0;
            int incl = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            if (i < n && bucket(i) == b) p.starts[i] = run + incl - c;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        for (int k = lane; k < (tot[b] + kTile - 1) / kTile; k += 32)
            reinterpret_cast<int4*>(p.tiles)[til[b] + k] =
                make_int4(b == adapters ? -1 : b, off[b] + kTile * k, min(kTile, tot[b] - kTile * k), 0);
    }
    __syncthreads();
    for (int i = warp; i < n; i += pool::kMetaThreads / 32) {
        const int c = count(i);
        if (c < kBig)
            for (int j = lane; j < c; j += 32) p.order[p.starts[i] + j] = lo(i) + j;
    }
    if (s_big)
        for (int i = 0; i < n; ++i) {
            const int c = count(i);
            if (c >= kBig)
                for (int j = threadIdx.x; j < c; j += pool::kMetaThreads) p.order[p.starts[i] + j] = lo(i) + j;
        }
}

// -- products ---------------------------------------------------------------------------------------
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
    const int n = on ? 16 : 0;                         // 0: fill with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct Args {
    const uint16_t *x, *y, *a, *b;
    uint16_t* out;
    const float* scale;
    float* part;                                       // [slices][total][R]; with one slice, h [total][R] bf16; few_kernel: slices 0, none
    const int32_t *head, *tiles, *order;
    int64_t x_stride, y_stride, out_stride;            // elements between rows
    int total, K, N, slices, k_per;                    // k_per: inputs of a slice, a multiple of kStep
    int cols;                                          // expand: column blocks of a CTA
};

constexpr int kStep = 128;                             // inputs of a stage
constexpr int kStages = 3;
constexpr int kShrinkWarps = 8;

// Row of `r` 16-byte chunks in shared memory, chunk index xor-ed with the row: ldmatrix without
// bank conflicts for rows of 128 bytes and more; for shorter rows several rows share 128 bytes.
template <int CH>
__device__ __forceinline__ uint32_t at(int row, int chunk) {
    if constexpr (CH >= 8) return (uint32_t)((row * CH + (chunk & ~7) + ((chunk ^ row) & 7)) * 16);
    else return (uint32_t)((row * CH + (chunk ^ ((row / (8 / CH)) & (CH - 1)))) * 16);
}

template <int R>
struct ShrinkSmem {
    static constexpr int kX = kTile * kStep * 2, kA = kStep * R * 2;
    static constexpr int kRing = kStages * (kX + kA);
    static constexpr int kRed = kShrinkWarps * 16 * R * 4;   // partial accumulators of the warps
    static constexpr int kBytes = kRing > kRed ? kRing : kRed;
};

// Inputs k0 .. k1 - 1 of tile t's x A, 4 sums at a time to store(index in [rows][R], sums).  Warps split
// the tile's 16-row blocks, and, where the tile has fewer than eight, the 16-input steps of a stage;
// those partial sums are added in warp order.
template <int R, class Store>
__device__ __forceinline__ void shrink_tile(const Args g, const int4 t, int k0, int k1, uint8_t* smem, Store store) {
    const int rows = t.z, first = t.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int steps = k1 > k0 ? (k1 - k0 + kStep - 1) / kStep : 0;
    const uint32_t base = sm100::smem_addr(smem);
    constexpr int XC = kStep / 8, AC = R / 8;          // chunks of a row
    constexpr int SZ = ShrinkSmem<R>::kX + ShrinkSmem<R>::kA;
    const uint16_t* A = g.a + (long)t.x * g.K * R;
    const int blocks = (rows + 15) / 16;
    const int mb = blocks <= 1 ? 1 : (blocks <= 2 ? 2 : 4);   // row blocks, rounded up; kw warps each
    const int kw = kShrinkWarps / mb;
    // this thread's x rows: chunk xc of rows xr, xr + XR, ...
    constexpr int XR = 32 * kShrinkWarps / XC, XN = kTile / XR;   // rows of a pass, passes
    const int xc = threadIdx.x % XC, xr = threadIdx.x / XC;
    const uint16_t* xrow[XN];
#pragma unroll
    for (int i = 0; i < XN; ++i) {
        const int r = xr + XR * i;
        xrow[i] = g.x + (r < rows ? (long)g.order[first + r] : 0) * g.x_stride + 8 * xc;
    }
    auto load = [&](int s) {
        if (s < steps) {
            const uint32_t st = base + (uint32_t)((s % kStages) * SZ);
            const int k = k0 + s * kStep;
#pragma unroll
            for (int i = 0; i < XN; ++i) {
                const int r = xr + XR * i;
                if (r < 16 * mb) {
                    const bool on = r < rows && k + 8 * xc < k1;
                    cp16(st + at<XC>(r, xc), on ? xrow[i] + k : g.x, on);
                }
            }
            for (int c = threadIdx.x; c < kStep * AC; c += 32 * kShrinkWarps) {
                const int kr = c / AC, cc = c % AC;
                const bool on = k + kr < k1;
                cp16(st + ShrinkSmem<R>::kX + at<AC>(kr, cc), on ? A + (long)(k + kr) * R + 8 * cc : g.a, on);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(s);
    float acc[R / 8][4];
#pragma unroll
    for (int j = 0; j < R / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    const int m = warp % mb, kk0 = warp / mb;
    for (int s = 0; s < steps; ++s) {
        cp_wait<kStages - 2>();
        __syncthreads();
        load(s + kStages - 1);
        const uint32_t st = base + (uint32_t)((s % kStages) * SZ);
        for (int kk = kk0; kk < kStep / 16; kk += kw) {
            uint32_t a[4];
            ldsm4(st + at<XC>(16 * m + (lane & 15), 2 * kk + (lane >> 4)), a);
#pragma unroll
            for (int j = 0; j < R / 16; ++j) {
                uint32_t b[4];
                ldsm4_t(st + ShrinkSmem<R>::kX + at<AC>(16 * kk + (lane & 15), 2 * j + (lane >> 4)), b);
                mma(acc[2 * j], a, b[0], b[1]);
                mma(acc[2 * j + 1], a, b[2], b[3]);
            }
        }
    }
    cp_wait<0>();
    __syncthreads();
    const int gq = lane >> 2, c = lane & 3;
    float* red = reinterpret_cast<float*>(smem);       // [kw][16 mb][R]
#pragma unroll
    for (int j = 0; j < R / 8; ++j) {
        float* p = red + (long)(kk0 * 16 * mb + 16 * m + gq) * R + 8 * j + 2 * c;
        *reinterpret_cast<float2*>(p) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(p + 8 * R) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    const int used = kw < kStep / 16 ? kw : kStep / 16;  // warps past a stage's steps hold zeros
    for (int i = threadIdx.x * 4; i < rows * R; i += 32 * kShrinkWarps * 4) {
        float4 v = *reinterpret_cast<const float4*>(red + i);
        for (int w = 1; w < used; ++w) {
            const float4 o = *reinterpret_cast<const float4*>(red + (long)w * 16 * mb * R + i);
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        store(i, v);
    }
}

// CTA (slice of the inputs, tile).
template <int R>
__global__ void __launch_bounds__(32 * kShrinkWarps)
shrink_kernel(const Args g) {
    extern __shared__ __align__(128) uint8_t smem[];
    // x, y and the plan are there, and this memory's last readers are done; from here on the expansion
    // may be brought in and fetch y and B
    grid_wait();
    grid_release();
    const int tile = blockIdx.y, slice = blockIdx.x;
    if (tile >= g.head[0]) return;
    const int4 t = reinterpret_cast<const int4*>(g.tiles)[tile];
    if (t.x < 0) return;
    const int k0 = slice * g.k_per, k1 = min(g.K, k0 + g.k_per);
    if (g.slices > 1) {
        float* dst = g.part + ((long)slice * g.total + t.y) * R;
        shrink_tile<R>(g, t, k0, k1, smem, [&](int i, const float4& v) { *reinterpret_cast<float4*>(dst + i) = v; });
    } else {
        uint16_t* h = reinterpret_cast<uint16_t*>(g.part) + (long)t.y * R;
        const float sc = g.scale != nullptr ? g.scale[t.x] : 1.f;
        shrink_tile<R>(g, t, k0, k1, smem, [&](int i, const float4& v) {
            *reinterpret_cast<uint2*>(h + i) = make_uint2(pack_bf16x2(v.x * sc, v.y * sc), pack_bf16x2(v.z * sc, v.w * sc));
        });
    }
}

constexpr int kExpandWarps = 4;                        // 32 columns each
constexpr int kBlockCols = 32 * kExpandWarps;          // columns of a block of the expansion

template <int R, int W>
struct ExpandSmem {
    static constexpr int kCols = 32 * W;               // columns of a block
    static constexpr int kH = kTile * R * 2, kB = R * kCols * 2, kY = kTile * kCols * 2;
    static constexpr int kBuf = kB + kY;
    static constexpr int kBytes = kH + 2 * kBuf;
};

// 8 values of h, scaled and rounded, to a tile's h in shared memory.
template <int R>
__device__ __forceinline__ void put_h(uint8_t* smem, int row, int chunk, const float (&v)[8], float sc) {
    *reinterpret_cast<uint4*>(smem + at<R / 8>(row, chunk)) =
        make_uint4(pack_bf16x2(v[0] * sc, v[1] * sc), pack_bf16x2(v[2] * sc, v[3] * sc),
                   pack_bf16x2(v[4] * sc, v[5] * sc), pack_bf16x2(v[6] * sc, v[7] * sc));
}

// y + h B of tile t in column blocks block0, block0 + skip, ... (n_blocks), staged in shared memory, the
// next block's y and B on their way meanwhile.  W warps; form() puts h (rows to the next multiple of 16,
// zeros past the tile's) at the start of `smem` once the first block is on its way.
template <int R, int W, class Form>
__device__ __forceinline__ void expand_tile(const Args g, const int4 t, uint8_t* smem, int block0, int skip, int n_blocks,
                                            Form form) {
    using S = ExpandSmem<R, W>;
    constexpr int kCols = S::kCols;
    const int rows = t.z, first = t.y;
    const bool copy_only = t.x < 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int YC = kCols / 8, HC = R / 8;
    constexpr int T = 32 * W, RS = T / YC, NR = kTile / RS;   // rows of a pass, passes
    const uint32_t sh = sm100::smem_addr(smem);
    const uint16_t* B = g.b + (long)(copy_only ? 0 : t.x) * R * g.N;
    const int c = threadIdx.x % YC, r0 = threadIdx.x / YC;      // this thread's chunk column, first row
    const int blocks = (rows + 15) / 16;
    int tok[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) tok[i] = r0 + i * RS < rows ? g.order[first + r0 + i * RS] : -1;
    // A thread copies in and writes out the same pieces of y, so a buffer's y needs no barrier between.
    auto load = [&](int blk) {
        if (blk < n_blocks) {
            const int col = (block0 + blk * skip) * kCols + 8 * c;
            const uint32_t sb = sh + S::kH + (blk & 1) * S::kBuf, sy = sb + S::kB;
            const bool on = col < g.N;
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (tok[i] >= 0) cp16(sy + at<YC>(r0 + i * RS, c), on ? g.y + tok[i] * g.y_stride + col : g.y, on);
            if (!copy_only)
#pragma unroll
                for (int k = 0; k < R / RS; ++k)
                    cp16(sb + at<YC>(r0 + k * RS, c), on ? B + (long)(r0 + k * RS) * g.N + col : g.b, on);
        }
        cp_commit();
    };
    load(0);
    form(sh, blocks);
    // h of the tile in registers for all blocks, where it fits (64 of a thread's at rank 64)
    constexpr bool kHeld = R <= 64;
    constexpr int MB = kTile / 16, KB = R / 16;
    uint32_t ha[kHeld ? MB : 1][KB][4];
    auto load_h = [&](int m, uint32_t (&a)[KB][4]) {
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) ldsm4(sh + at<HC>(16 * m + (lane & 15), 2 * kk + (lane >> 4)), a[kk]);
    };
    if (kHeld && !copy_only) {
        __syncthreads();
#pragma unroll
        for (int m = 0; m < (kHeld ? MB : 1); ++m)
            if (m < blocks) load_h(m, ha[m]);
    }
    for (int blk = 0; blk < n_blocks; ++blk) {
        load(blk + 1);
        cp_wait<1>();
        __syncthreads();
        const uint32_t sb = sh + S::kH + (blk & 1) * S::kBuf;
        uint8_t* yb = smem + S::kH + (blk & 1) * S::kBuf + S::kB;
        if (!copy_only) {
            const int gq = lane >> 2, cq = lane & 3;
            constexpr int CJ = kCols / W / 16;   // 16-column pieces of a warp
            uint32_t b[KB][CJ][4];                     // B of this warp's columns, for every row block
#pragma unroll
            for (int kk = 0; kk < KB; ++kk)
#pragma unroll
                for (int j = 0; j < CJ; ++j)
                    ldsm4_t(sb + at<YC>(16 * kk + (lane & 15), 2 * (CJ * warp + j) + (lane >> 4)), b[kk][j]);
            auto rows16 = [&](int m, const uint32_t (&a)[KB][4]) {
                float acc[2 * CJ][4] = {};
#pragma unroll
                for (int kk = 0; kk < KB; ++kk)
#pragma unroll
                    for (int j = 0; j < CJ; ++j) {
                        mma(acc[2 * j], a[kk], b[kk][j][0], b[kk][j][1]);
                        mma(acc[2 * j + 1], a[kk], b[kk][j][2], b[kk][j][3]);
                    }
#pragma unroll
                for (int j = 0; j < 2 * CJ; ++j)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {   // rows past the tile's are scratch
                        const int r = 16 * m + gq + 8 * half;
                        uint32_t* p = reinterpret_cast<uint32_t*>(yb + at<YC>(r, 2 * CJ * warp + j)) + cq;
                        const uint32_t w = *p;
                        *p = pack_bf16x2(bf16lo_to_f32(w) + acc[j][2 * half], bf16hi_to_f32(w) + acc[j][2 * half + 1]);
                    }
            };
            if constexpr (kHeld) {
#pragma unroll
                for (int m = 0; m < MB; ++m)
                    if (m < blocks) rows16(m, ha[m]);
            } else {
                for (int m = 0; m < blocks; ++m) {
                    uint32_t a[KB][4];
                    load_h(m, a);
                    rows16(m, a);
                }
            }
            __syncthreads();
        }
        const int col = (block0 + blk * skip) * kCols + 8 * c;
        if (col < g.N) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                if (tok[i] >= 0)
                    *reinterpret_cast<uint4*>(g.out + tok[i] * g.out_stride + col) =
                        *reinterpret_cast<const uint4*>(yb + at<YC>(r0 + i * RS, c));
        }
    }
}

// CTA (group of column blocks, tile).
template <int R>
__global__ void __launch_bounds__(32 * kExpandWarps)
expand_kernel(const Args g) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kCols = ExpandSmem<R, kExpandWarps>::kCols, HC = R / 8, T = 32 * kExpandWarps;
    const int tile = blockIdx.y;
    const bool none = tile >= g.head[0];
    const int4 t = none ? make_int4(-1, 0, 0, 0) : reinterpret_cast<const int4*>(g.tiles)[tile];
    if (none || (t.x < 0 && g.y == g.out)) {
        grid_wait();
        return;
    }
    const int block0 = blockIdx.x * g.cols;
    const int n_blocks = min(g.cols, (g.N + kCols - 1) / kCols - block0);
    expand_tile<R, kExpandWarps>(g, t, smem, block0, 1, n_blocks, [&](uint32_t, int blocks) {
        const int rows = t.z, first = t.y;
        const bool copy_only = t.x < 0;
        grid_wait();                                                // h is there
        if (!copy_only) {
            if (g.slices == 1) {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(g.part) + (long)first * R;
                for (int i = threadIdx.x; i < 16 * blocks * HC; i += T) {
                    const int r = i / HC, ch = i % HC;
                    *reinterpret_cast<uint4*>(smem + at<HC>(r, ch)) =
                        r < rows ? *reinterpret_cast<const uint4*>(h + (long)r * R + 8 * ch) : make_uint4(0, 0, 0, 0);
                }
            } else {                                       // partials summed in slice order, scaled, rounded
                const float sc = g.scale != nullptr ? g.scale[t.x] : 1.f;
                for (int i = threadIdx.x; i < 16 * blocks * HC; i += T) {
                    const int r = i / HC, ch = i % HC;
                    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (r < rows) {
#pragma unroll 4
                        for (int s = 0; s < g.slices; ++s) {
                            const float4* p = reinterpret_cast<const float4*>(g.part + ((long)s * g.total + first + r) * R + 8 * ch);
                            const float4 a = p[0], b = p[1];
                            v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                            v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
                        }
                    }
                    put_h<R>(smem, r, ch, v, sc);
                }
            }
        }
    });
}

// A decode batch's tiles (a few rows each): a cluster of kParts CTAs a tile, in one launch and without a
// workspace (96 rows of 16 adapters, 4096 -> 6144, rank 16: 19.7 us a call, plan included, 24.1 in two).  Each CTA sums a
// slice of the inputs; the sums are exchanged through distributed shared memory, added in slice order by
// every CTA, and the column blocks shared out.
constexpr int kParts = 8;                              // portable cluster size
// kAhead: with an SM to itself a CTA has memory of its own for the column blocks, and the first is on its way
// during the sums (5 tiles, 4096 -> 6144, rank 16: 12.3 us, 14.3 without).  For up to half of the SMs: clusters
// of 8 such CTAs do not cover them all (18 tiles, 4096 -> 28672: 36.9 us, 24.6 without).
template <int R, bool kAhead>
struct FewSmem {
    static constexpr int kRing = kTile * R * 4;        // before it this CTA's sums [row][R]
    static constexpr int kShrink = ShrinkSmem<R>::kBytes, kExpand = ExpandSmem<R, kShrinkWarps>::kBytes;
    static constexpr int kBlocks = kRing + (kAhead ? kShrink : 0);
    static constexpr int kBytes = kAhead || kExpand > kShrink ? kBlocks + kExpand : kRing + kShrink;
};
template <int R, bool kAhead>
__global__ void __launch_bounds__(32 * kShrinkWarps)
few_kernel(const Args g) {
    using S = FewSmem<R, kAhead>;
    extern __shared__ __align__(128) uint8_t smem[];
    grid_wait();
    grid_release();
    const int tile = blockIdx.x / kParts, slice = blockIdx.x % kParts;
    if (tile >= g.head[0]) return;                     // (the whole cluster, here and below)
    const int4 t = reinterpret_cast<const int4*>(g.tiles)[tile];
    if (t.x < 0 && g.y == g.out) return;
    cg::cluster_group cluster = cg::this_cluster();
    float* part = reinterpret_cast<float*>(smem);
    uint8_t* rest = smem + S::kBlocks;
    auto sums = [&]() {
        const int k0 = slice * g.k_per, k1 = min(g.K, k0 + g.k_per);
        shrink_tile<R>(g, t, k0, k1, smem + S::kRing, [&](int i, const float4& v) { *reinterpret_cast<float4*>(part + i) = v; });
    };
    if (!kAhead && t.x >= 0) {
        sums();
        __syncthreads();                               // `rest` is free
    }
    constexpr int kCols = ExpandSmem<R, kShrinkWarps>::kCols, HC = R / 8;
    const int all = (g.N + kCols - 1) / kCols, n_blocks = all > slice ? (all - slice + kParts - 1) / kParts : 0;
    expand_tile<R, kShrinkWarps>(g, t, rest, slice, kParts, n_blocks, [&](uint32_t, int blocks) {
        if (t.x < 0) return;
        const float sc = g.scale != nullptr ? g.scale[t.x] : 1.f;
        if (kAhead) sums();
        cluster.sync();
        for (int i = threadIdx.x; i < 16 * blocks * HC; i += 32 * kShrinkWarps) {
            const int r = i / HC, ch = i % HC;
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (r < t.z) {
                float4 x[kParts][2];
#pragma unroll
                for (int s = 0; s < kParts; ++s) {
                    const float4* p = reinterpret_cast<const float4*>(cluster.map_shared_rank(part + r * R + 8 * ch, s));
                    x[s][0] = p[0];
                    x[s][1] = p[1];
                }
#pragma unroll
                for (int s = 0; s < kParts; ++s) {
                    v[0] += x[s][0].x; v[1] += x[s][0].y; v[2] += x[s][0].z; v[3] += x[s][0].w;
                    v[4] += x[s][1].x; v[5] += x[s][1].y; v[6] += x[s][1].z; v[7] += x[s][1].w;
                }
            }
            put_h<R>(rest, r, ch, v, sc);
        }
        cluster.sync();                                // others may still read this CTA's sums
    });
}

// Whether one launch of clusters does it (few_kernel).  Its CTAs fill three quarters of the SMs at least,
// and two fit each (14 tiles, 4096 -> 28672, rank 16: 22.5 us against 26.6 in two launches; 10 tiles 22.5 :
// 20.5; 19 tiles, 4096 -> 6144, rank 16 14.3 : 16.4, 32 16.4 : 18.4, 64 26.7 : 20.5); or the work is
// small enough for fewer (1 to 10 tiles of rank 16, up to 8192 wide, a few rows each: 10 to 12 us both, and a
// launch and a workspace less for the host: 4 us).
inline bool is_few(int total, int n, int adapters, int inputs, int outputs, int rank, int sms) {
    const long tiles = max_tiles(total, n, adapters), ctas = tiles * kParts;
    if (rank > 32 || ctas > 2L * sms) return false;
    return 4 * ctas >= 3L * sms || (rank == 16 && inputs <= 8192 && outputs <= 8192 && total <= 16 * tiles);
}

inline int slices_for(int total, int n, int adapters, int K, int sms) {
    // Slices of the inputs, 256 at least, until the CTAs are one and a half per SM (two fit on an SM).
    const long tiles = max_tiles(total, n, adapters);
    int s = 1;
    while (s < 32 && 2 * tiles * s < 3L * sms && K >= 2 * s * 256) s *= 2;
    return s;
}

// Column blocks of a CTA: as many as leave about four waves of resident CTAs (h is formed once for
// them; fewer, longer CTAs end less evenly).
inline int column_blocks(int blocks, int tiles, int rank, int sms) {
    const long bytes = 128L * rank + 2L * (256L * rank + 16384) + 1024;   // shared memory of a CTA
    const long slots = sms * std::max(1L, std::min(8L, 233472L / bytes));
    return (int)std::max(1L, std::min(32L, (long)blocks * tiles / (4 * slots)));
}

template <int R>
static int launch(const Args& g, int tiles, int sms, cudaStream_t st) {
    static PerContextOnce once;
    const int rc = once.run([] {
        LF_CHECK_CUDA(cudaFuncSetAttribute(shrink_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           ShrinkSmem<R>::kBytes));
        LF_CHECK_CUDA(cudaFuncSetAttribute(expand_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           ExpandSmem<R, kExpandWarps>::kBytes));
        if constexpr (R <= 32) {
            LF_CHECK_CUDA(cudaFuncSetAttribute((few_kernel<R, true>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               FewSmem<R, true>::kBytes));
            LF_CHECK_CUDA(cudaFuncSetAttribute((few_kernel<R, false>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               FewSmem<R, false>::kBytes));
        }
        return LF_OK;
    });
    if (rc != LF_OK) return rc;
    if constexpr (R <= 32) {
        const dim3 grid((unsigned)(tiles * kParts)), block(32 * kShrinkWarps);
        if (g.slices == 0)
            return 2 * tiles * kParts <= sms
                       ? launch_early_clusters("lora", few_kernel<R, true>, kParts, grid, block, FewSmem<R, true>::kBytes, st, g)
                       : launch_early_clusters("lora", few_kernel<R, false>, kParts, grid, block, FewSmem<R, false>::kBytes, st, g);
    }
    const int e = launch_early("lora shrink", shrink_kernel<R>, dim3(g.slices, tiles), dim3(32 * kShrinkWarps),
                               ShrinkSmem<R>::kBytes, st, g);
    if (e != LF_OK) return e;
    return launch_early("lora expand", expand_kernel<R>, dim3(((g.N + kBlockCols - 1) / kBlockCols + g.cols - 1) / g.cols, tiles),
                        dim3(32 * kExpandWarps), ExpandSmem<R, kExpandWarps>::kBytes, st, g);
}

static int sm_count(int* out) {
    int dev = 0;
    LF_CHECK_CUDA(cudaGetDevice(&dev));
    LF_CHECK_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return LF_OK;
}

static int check_sizes(int n, int total, int adapters) {
    LF_CHECK_ARG(n >= 0 && total >= 0, "lora: negative sizes");
    LF_CHECK_ARG(adapters > 0 && adapters <= kMaxAdapters, "lora: 1..%d adapters", kMaxAdapters);
    LF_CHECK_ARG(n > 0 || total == 0, "lora: tokens without sessions");
    LF_CHECK_ARG(total <= 64 * 60000, "lora: too many tokens");
    return LF_OK;
}

}  // namespace lora
}  // namespace lf

using namespace lf;

extern "C" int lf_lora_plan_size(int n, int total_tokens, int num_adapters, size_t* bytes) {
    LF_CHECK_ARG(bytes != nullptr, "lora plan: bytes is null");
    const int rc = lora::check_sizes(n, total_tokens, num_adapters);
    if (rc != LF_OK) return rc;
    *bytes = 4 * (size_t)(lora::kHeader + 4 * lora::max_tiles(total_tokens, n, num_adapters) + total_tokens + n);
    clear_error();
    return LF_OK;
}

extern "C" int lf_lora_plan(const int32_t* adapter_ids, const int32_t* cu_tokens, int n, int total_tokens,
                            int num_adapters, void* plan, size_t plan_bytes, void* stream) {
    size_t need = 0;
    int rc = lf_lora_plan_size(n, total_tokens, num_adapters, &need);
    if (rc != LF_OK) return rc;
    LF_CHECK_ARG(plan != nullptr && aligned16(plan) && plan_bytes >= need, "lora plan: needs %zu bytes, 16-byte aligned", need);
    LF_CHECK_ARG(n == 0 || (adapter_ids && cu_tokens), "lora plan: null pointer argument");
    static PerContextOnce once;
    rc = once.run([] {
        LF_CHECK_CUDA(cudaFuncSetAttribute(lora::plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           3 * (lora::kMaxAdapters + 1) * 4));
        return LF_OK;
    });
    if (rc != LF_OK) return rc;
    const lora::Plan p = lora::views(static_cast<int32_t*>(plan), total_tokens, n, num_adapters);
    return launch_early("lora plan", lora::plan_kernel, dim3(1), dim3(pool::kMetaThreads), 3 * (num_adapters + 1) * 4,
                        (cudaStream_t)stream, adapter_ids, cu_tokens, n, total_tokens, num_adapters, p);
}

extern "C" int lf_lora_workspace_size(int n, int total_tokens, int num_adapters, int inputs, int outputs,
                                      int rank, int sm_count, size_t* bytes) {
    LF_CHECK_ARG(bytes != nullptr, "lora: bytes is null");
    int rc = lora::check_sizes(n, total_tokens, num_adapters);
    if (rc != LF_OK) return rc;
    LF_CHECK_ARG(inputs > 0 && outputs > 0 && rank > 0, "lora: bad workspace arguments");
    if (sm_count <= 0) {
        rc = lora::sm_count(&sm_count);
        if (rc != LF_OK) return rc;
    }
    *bytes = lora::is_few(total_tokens, n, num_adapters, inputs, outputs, rank, sm_count)
                 ? 0 : (size_t)lora::slices_for(total_tokens, n, num_adapters, inputs, sm_count) * total_tokens * rank * 4;
    clear_error();
    return LF_OK;
}

extern "C" int lf_lora_add(const lf_bf16* y, int64_t y_stride, const lf_bf16* x, int64_t x_stride,
                           const lf_bf16* a, const lf_bf16* b, const float* scale, const void* plan, int n,
                           int total_tokens, int num_adapters, int inputs, int outputs, int rank,
                           lf_bf16* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
                           int sm_count, void* stream) {
    int rc = lora::check_sizes(n, total_tokens, num_adapters);
    if (rc != LF_OK) return rc;
    LF_CHECK_ARG(rank == 16 || rank == 32 || rank == 64 || rank == 128,
                 "lora: rank must be 16, 32, 64 or 128 (got %d; pad A and B with zeros)", rank);
    LF_CHECK_ARG(inputs > 0 && inputs % 8 == 0 && outputs > 0 && outputs % 8 == 0,
                 "lora: inputs and outputs must be positive multiples of 8");
    if (total_tokens == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(y && x && a && b && plan && out, "lora: null pointer argument");
    LF_CHECK_ARG(aligned16(y) && aligned16(x) && aligned16(a) && aligned16(b) && aligned16(out) &&
                     aligned16(plan) && aligned16(workspace) && y_stride % 8 == 0 && x_stride % 8 == 0 &&
                     out_stride % 8 == 0,
                 "lora: rows must be 16-byte aligned");
    LF_CHECK_ARG(total_tokens == 1 || (y_stride >= outputs && out_stride >= outputs && x_stride >= 0),
                 "lora: rows of y or out overlap");
    LF_CHECK_ARG(y != out || y_stride == out_stride, "lora: in place, y and out need the same rows");
    if (sm_count <= 0) {
        rc = lora::sm_count(&sm_count);
        if (rc != LF_OK) return rc;
    }
    lora::Args g{};
    const bool few = lora::is_few(total_tokens, n, num_adapters, inputs, outputs, rank, sm_count);
    g.slices = few ? 0 : lora::slices_for(total_tokens, n, num_adapters, inputs, sm_count);
    const size_t need = (size_t)g.slices * total_tokens * rank * 4;
    LF_CHECK_ARG(workspace != nullptr || need == 0, "lora: null pointer argument");
    LF_CHECK_ARG(workspace_bytes >= need, "lora: workspace too small (%zu < %zu bytes)", workspace_bytes, need);
    const lora::Plan p = lora::views(const_cast<int32_t*>(static_cast<const int32_t*>(plan)), total_tokens, n, num_adapters);
    g.x = x;
    g.y = y;
    g.a = a;
    g.b = b;
    g.out = out;
    g.scale = scale;
    g.part = static_cast<float*>(workspace);
    g.head = p.head;
    g.tiles = p.tiles;
    g.order = p.order;
    g.x_stride = x_stride;
    g.y_stride = y_stride;
    g.out_stride = out_stride;
    g.total = total_tokens;
    g.K = inputs;
    g.N = outputs;
    const int steps = (inputs + lora::kStep - 1) / lora::kStep;
    const int cuts = few ? lora::kParts : g.slices;
    g.k_per = (steps + cuts - 1) / cuts * lora::kStep;
    const int tiles = (int)lora::max_tiles(total_tokens, n, num_adapters);
    g.cols = lora::column_blocks((outputs + lora::kBlockCols - 1) / lora::kBlockCols, tiles, rank, sm_count);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (rank) {
        case 16: return lora::launch<16>(g, tiles, sm_count, st);
        case 32: return lora::launch<32>(g, tiles, sm_count, st);
        case 64: return lora::launch<64>(g, tiles, sm_count, st);
        default: return lora::launch<128>(g, tiles, sm_count, st);
    }
}
