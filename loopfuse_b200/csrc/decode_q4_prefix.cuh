// The shared prefix of the 4-bit decode on the tcgen05 tensor cores: for batches with enough query
// rows (sessions x heads of a group) to use tiles of 128.
//
// A CTA takes (chunk of the prefix, KV head, tile of 128 query rows), in steps of 32 tokens (2 pages).
// What a softmax thread, which owns a row, would have to do for each token's two scales and lows is left
// to the tensor cores, which have the time.  s n (12 bits) is the exact sum of two bf16 values,
// h = bf16(s n) and s n - h, and so is s (n - 8), so that with B = low + 8 s
//   q . k = sum of q (h_k + l_k) + low sum(q)           low is bf16; sum(q) goes in as three bf16 parts
//   o     = sum of bf16(p) (h_v + l_v) + p B            the last with unrounded p, in the softmax threads
// As in decode_q4.cu the only rounding to fewer bits is that of the probabilities that multiply s (n - 8).
//
//   unpack   4 warps write the pages' h and l as 128-byte swizzled tiles, B in fp32.
//   MMA      one thread issues S = Q . K^T, Q in tensor memory, and, a step behind, O += P . V.
//   softmax  4 warps, a thread a row: an online maximum (raised only when it grows by more than 8 in
//            log2 units, so that O is seldom rescaled), fp32 sums, P written over S.
//
// Tensor memory: O, two buffers of S (P takes a buffer's first columns), Q: 256 columns, so that two
// CTAs fit an SM.  A NaN among a token's scales must not reach rows that do not hold the token: its tile
// of V is then zero and B brings the NaN, behind the row's mask.
//
// 64 sessions x 4 heads a KV head on 4096 tokens: the whole decode takes 45.3 us, 52.7 with the warp-MMA
// form; 256 sessions: 81 and 146.  What bounds it: a step's chain unpack - S - softmax - P . V, 2400
// cycles for the two CTAs of an SM together, half of that the softmax's and unpacking's instructions, and
// about 10 us around the 8 steps of a CTA (first pages and code from HBM, partials written).  Measured
// and not kept, same case when it took 43.4: scales applied by the softmax threads (S of each group apart: two 16-byte
// shared loads a token and row) 51.1; pages through a ring of bulk copies 45.8; one CTA an SM with twice
// the steps 47.3; chunks merged over clusters of 8 CTAs 46.0; one softmax body, masked always, 46.2.
// Waits are bounded (sites 255..259 in the device error word); after one gives up every role leaves.
#pragma once

#include "q4_common.cuh"
#include "sm100_primitives.cuh"

namespace lf {
namespace q4 {

constexpr int kTcRows = 128;                           // query rows of a tile
constexpr int kTcPages = 2;                            // pages of a step
constexpr int kTcKeys = kTcPages * kPage;
constexpr int kTcThreads = 288;                        // softmax 0-3, unpack 4-7, MMA 8
constexpr int kTcPerSm = 2;

template <int D>
struct TcSmem {
    static constexpr int NG = Fmt<D>::NG;
    static constexpr int kTile = kTcKeys * 128;        // 64 dims of a step's tokens
    static constexpr int kHalf = NG * kTile;           // h or l of a step
    static constexpr int kQs = 0;                      // [row][128 bytes]: parts of sum(q), 16 slots in use
    static constexpr int kK = kTcRows * 128;           // [buffer][h, l][group]
    static constexpr int kV = kK + 4 * kHalf;          // [buffer][group][h, l]
    static constexpr int kLow = kV + 4 * kHalf;        // [buffer][token][128 bytes]: lows, 16 slots in use
    static constexpr int kB = kLow + 2 * kTile;        // [buffer][token] float2: B of V's groups
    static constexpr int kBytes = kB + 2 * kTcKeys * 8 + 1024;
};

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The codes at bits 0..3 of both halves, as bf16 128 + n.
__device__ __forceinline__ uint32_t codes128(uint32_t w) {
    uint32_t n;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(n) : "r"(w), "n"(0x000F000F), "r"(0x43004300u));
    return n;
}
// c s = h + l exactly (c of 4 bits, s of 8).
__device__ __forceinline__ void split_product(uint32_t c, uint32_t s, uint32_t& h, uint32_t& l) {
    asm("{\n\t.reg .b32 m;\n\t"
        "mul.rn.bf16x2 %0, %2, %3;\n\t"
        "neg.bf16x2 m, %0;\n\t"
        "fma.rn.bf16x2 %1, %2, %3, m;\n\t}"
        : "=&r"(h), "=r"(l) : "r"(c), "r"(s));
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, kTcPerSm) prefix_tc_kernel(const DecodeArgs a) {
    using namespace sm100;
    using F = Fmt<D>;
    using S = TcSmem<D>;
    constexpr int NG = F::NG, NW = 2 * NG;
    constexpr int kS = D, kQ = kS + 2 * kTcKeys, kCols = 256;   // tensor memory columns; O at 0
    static_assert(kQ + D / 2 <= kCols, "tensor memory");
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t q_full, kv_full[2], kv_free[2], s_full[2], p_full[2], o_full[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int err;
    grid_wait();
    grid_release();                                    // the own pages need nothing from here
    const int chunk = blockIdx.x % a.n_chunks, h = blockIdx.x / a.n_chunks % a.Hkv;
    const int tile = blockIdx.x / a.n_chunks / a.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = a.N * a.G, row0 = tile * kTcRows;
    const int p_begin = chunk * a.chunk, p_end = min(p_begin + a.chunk, a.n_prefix);
    // The page ids come from the tile's longest session, whose row holds every page that any session
    // here needs; pages past its length are not read.
    int best = -1, lead = row0 / a.G;
    for (int n = row0 / a.G + lane; n <= min(row0 + kTcRows - 1, rows - 1) / a.G; n += 32) {
        const int L = held(a, n);
        if (L > best) { best = L; lead = n; }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const int ob = __shfl_xor_sync(0xffffffffu, best, off), ol = __shfl_xor_sync(0xffffffffu, lead, off);
        if (ob > best || (ob == best && ol < lead)) { best = ob; lead = ol; }
    }
    const int pages = min(p_end, (best + kPage - 1) / kPage) - p_begin;
    if (pages <= 0) return;                            // (the whole CTA) combine reads no slot of this chunk
    const int steps = (pages + kTcPages - 1) / kTcPages;

    if (warp == 8) {
        if (lane == 0) {
            mbar_init(smem_addr(&q_full), 128);
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_addr(&kv_full[b]), 128);
                mbar_init(smem_addr(&kv_free[b]), 1);
                mbar_init(smem_addr(&s_full[b]), 1);
                mbar_init(smem_addr(&p_full[b]), 128);
                mbar_init(smem_addr(&o_full[b]), 1);
            }
            mbar_init(smem_addr(&drained), 1);
            err = 0;
            fence_barrier_init();
        }
        __syncwarp();
        tmem_alloc(smem_addr(&tmem_slot), kCols);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, sbase = smem_addr(smem);
    auto wait = [&](uint64_t& bar, int phase, int site) {      // warp-uniform answer
        return __all_sync(0xffffffffu, mbar_wait(smem_addr(&bar), (uint32_t)(phase & 1), &err, site));
    };

    if (warp < 4) {
        // ---- softmax: thread = query row = tensor memory lane ----
        const int r = threadIdx.x, row = row0 + r;
        const bool live = row < rows;
        const int n = row / a.G;
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        {                                              // Q and the parts of its sums
            const uint16_t* q = a.q + ((size_t)n * a.Hq + h * a.G + row % a.G) * D;
            uint32_t part[4] = {0, 0, 0, 0};           // h0 m0 l0 h1 m1 l1 - -
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float sum = 0.f;
                uint32_t x[32];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (live) y = *reinterpret_cast<const uint4*>(q + g * 64 + j * 8);
                    const uint32_t w[4] = {y.x ^ a.flip, y.y ^ a.flip, y.z ^ a.flip, y.w ^ a.flip};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        x[4 * j + k] = w[k];
                        sum += bf16lo_to_f32(w[k]) + bf16hi_to_f32(w[k]);
                    }
                }
                tmem_st32(lanes + (uint32_t)(kQ + 32 * g), x);
                const uint32_t hi = pack_bf16x2(sum, 0.f);
                const float r1 = sum - bf16lo_to_f32(hi);
                const uint32_t mid = pack_bf16x2(r1, 0.f);
                const uint32_t low = pack_bf16x2(r1 - bf16lo_to_f32(mid), 0.f);
                if (g == 0) {
                    part[0] = (hi & 0xFFFFu) | mid << 16;
                    part[1] = low & 0xFFFFu;
                } else {
                    part[1] |= hi << 16;
                    part[2] = (mid & 0xFFFFu) | low << 16;
                }
            }
            auto slot = [&](int ch) { return reinterpret_cast<uint4*>(smem + S::kQs + r * 128 + ((ch ^ (r & 7)) << 4)); };
            *slot(0) = make_uint4(part[0], part[1], part[2], part[3]);
            *slot(1) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_addr(&q_full));
        }
        const int end = (p_begin + pages) * kPage;     // a step's missing page is past it
        const int len = live ? min(end, held(a, n)) : 0;
        int lmin = live ? len : 0x7FFFFFFF;            // rows past the batch are not stored: any mask will do
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) lmin = min(lmin, __shfl_xor_sync(0xffffffffu, lmin, off));
        lmin = min(lmin, end);
        const float qscale = a.qscale / kDown;         // scores here are q . k themselves
        uint64_t bias2 = 0;                            // sum p B, per group
        uint64_t l2 = 0;                               // sum p, even and odd tokens
        float m = -INFINITY;
        bool ok = true;
        auto step = [&](int i, auto masked) {
            constexpr bool kMasked = decltype(masked)::value;
            const int b = i & 1, tok0 = p_begin * kPage + i * kTcKeys;
            const float2* B = reinterpret_cast<const float2*>(smem + S::kB) + b * kTcKeys;
            const uint32_t ts = lanes + (uint32_t)(kS + b * kTcKeys);
            uint32_t x[kTcKeys];
            tmem_ld32(ts, x);
            tmem_wait_ld();
            float s[kTcKeys], mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < kTcKeys; ++k) {
                s[k] = __uint_as_float(x[k]);
                if (kMasked) s[k] = tok0 + k < len ? s[k] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < kTcKeys; k += 2) mx = fmax3(mx, s[k], s[k + 1]);
            const bool grow = m == -INFINITY ? mx > -INFINITY : (mx - m) * qscale > 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float to = grow ? mx : m;
                const float f = m == -INFINITY ? 0.f : (m == to ? 1.f : fast_exp2((m - to) * qscale));
                m = to;
                const float2 bb = f2_unpack(bias2), ll = f2_unpack(l2);
                bias2 = f2_pack(bb.x * f, bb.y * f);
                l2 = f2_pack(ll.x * f, ll.y * f);
                if (i > 0) {                           // O holds the steps before: rescale it in place
                    if (!wait(o_full[(i - 1) & 1], (i - 1) >> 1, 258)) return false;
                    tc_fence_after();
#pragma unroll 1
                    for (int cc = 0; cc < D / 32; ++cc) {
                        uint32_t o[32];
                        tmem_ld32(lanes + (uint32_t)(cc * 32), o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st32(lanes + (uint32_t)(cc * 32), o);
                    }
                    tmem_wait_st();
                }
            }
            const float ref = m == -INFINITY ? 0.f : m * -qscale;
            const uint64_t qs2 = f2_pack(qscale, qscale), ref2 = f2_pack(ref, ref);
            uint32_t p[kTcKeys / 2];
#pragma unroll
            for (int k = 0; k < kTcKeys; k += 2) {
                const float2 t = f2_unpack(ffma2(f2_pack(s[k], s[k + 1]), qs2, ref2));
                float e0 = fast_exp2(t.x), e1 = fast_exp2(t.y);
                const float4 bb = *reinterpret_cast<const float4*>(B + k);
                if (kMasked) {                         // what a masked token's scales hold does not count
                    const bool keep0 = tok0 + k < len, keep1 = tok0 + k + 1 < len;
                    e0 = keep0 ? e0 : 0.f;
                    e1 = keep1 ? e1 : 0.f;
                    if (keep0) bias2 = ffma2(f2_pack(e0, e0), f2_pack(bb.x, bb.y), bias2);
                    if (keep1) bias2 = ffma2(f2_pack(e1, e1), f2_pack(bb.z, bb.w), bias2);
                } else {
                    bias2 = ffma2(f2_pack(e0, e0), f2_pack(bb.x, bb.y), bias2);
                    bias2 = ffma2(f2_pack(e1, e1), f2_pack(bb.z, bb.w), bias2);
                }
                l2 = fadd2(l2, f2_pack(e0, e1));
                p[k / 2] = pack_bf16x2(e0, e1);
            }
#pragma unroll
            for (int k = 0; k < kTcKeys / 2; k += 8)
                tmem_st8(ts + (uint32_t)k, {p[k], p[k + 1], p[k + 2], p[k + 3], p[k + 4], p[k + 5], p[k + 6], p[k + 7]});
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_addr(&p_full[b]));
            return true;
        };
        for (int i = 0; i < steps && ok; ++i) {
            // (kv_full, long complete, for what the unpack warps wrote to B)
            ok = wait(s_full[i & 1], i >> 1, 257) && wait(kv_full[i & 1], i >> 1, 257);
            if (!ok) break;
            tc_fence_after();
            if ((p_begin + (i + 1) * kTcPages) * kPage <= lmin) ok = step(i, std::false_type{});
            else ok = step(i, std::true_type{});
        }
        if (ok) ok = wait(o_full[(steps - 1) & 1], (steps - 1) >> 1, 258);
        if (ok) {
            tc_fence_after();
            // Through shared memory (K and V are done with), so that a warp stores whole rows; 16-byte
            // pieces of a row are rotated by its number.
            const float2 bb = f2_unpack(bias2), ll = f2_unpack(l2);
            float4* stage = reinterpret_cast<float4*>(smem + S::kK) + warp * 32 * (D / 4);
#pragma unroll
            for (int cc = 0; cc < D / 32; ++cc) {
                uint32_t o[32];
                tmem_ld32(lanes + (uint32_t)(cc * 32), o);
                tmem_wait_ld();
                const float add = cc < 2 ? bb.x : bb.y;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    stage[lane * (D / 4) + ((cc * 8 + k + lane) & (D / 4 - 1))] =
                        make_float4(__uint_as_float(o[4 * k]) + add, __uint_as_float(o[4 * k + 1]) + add,
                                    __uint_as_float(o[4 * k + 2]) + add, __uint_as_float(o[4 * k + 3]) + add);
            }
            __syncwarp();
            constexpr int kLanes = D / 4;              // lanes of a row
#pragma unroll 8
            for (int k = 0; k < 32; k += 32 / kLanes) {
                const int r2 = k + lane / kLanes, row2 = row0 + warp * 32 + r2, piece = lane % kLanes;
                const size_t slot = ((size_t)(row2 / a.G) * a.Hq + h * a.G + row2 % a.G) * a.n_chunks + chunk;
                if (row2 < rows)
                    reinterpret_cast<float4*>(a.pre_o + slot * D)[piece] = stage[r2 * (D / 4) + ((piece + r2) & (D / 4 - 1))];
            }
            const size_t slot = ((size_t)n * a.Hq + h * a.G + row % a.G) * a.n_chunks + chunk;
            if (live) a.pre_ml[slot] = make_float2(m / kDown, ll.x + ll.y);   // the other pieces' units
            tc_fence_before();
        }
    } else if (warp < 8) {
        // ---- unpack: warp = 8 tokens of the step, half a page ----
        const int w = warp - 4, page_i = w >> 1, half = w & 1, g = lane >> 2, c = lane & 3;
        const int32_t* row = a.bt + (size_t)lead * a.max_pages + p_begin;
        struct Raw { uint32_t k[NW], v[NW], pk[NW], pv[2][NG]; };   // pk: token g; pv: tokens 2c, 2c + 1
        auto page_of = [&](int i) {
            const int k = i * kTcPages + page_i;
            return k < pages ? checked_page(row[k], a.num_pages) : -1;
        };
        auto get4 = [](const uint8_t* p, uint32_t* d) {
            const uint4 t = *reinterpret_cast<const uint4*>(p);
            d[0] = t.x; d[1] = t.y; d[2] = t.z; d[3] = t.w;
        };
        auto get2 = [](const uint8_t* p, uint32_t* d) {
            const uint2 t = *reinterpret_cast<const uint2*>(p);
            d[0] = t.x; d[1] = t.y;
        };
        auto load = [&](int page, Raw& x) {            // zeros for a page past the chunk
            if (page < 0) {
#pragma unroll
                for (int j = 0; j < NW; ++j) x.k[j] = x.v[j] = x.pk[j] = x.pv[j / NG][j % NG] = 0;
                return;
            }
            const uint8_t* blk = a.pages + ((size_t)page * a.Hkv + h) * F::kBlockBytes;
            const uint8_t* par = blk + F::kParOff + half * 8 * (8 * NG);
            if constexpr (NG == 2) {
                get4(blk + (half * 8 + g) * 64 + c * 16, x.k);
                get4(blk + F::kVOff + half * 512 + lane * 16, x.v);
                get4(par + g * 16, x.pk);
                get2(par + 2 * c * 16 + 8, x.pv[0]);
                get2(par + (2 * c + 1) * 16 + 8, x.pv[1]);
            } else {
                get2(blk + (half * 8 + g) * 32 + c * 8, x.k);
                get2(blk + F::kVOff + half * 256 + lane * 8, x.v);
                get2(par + g * 8, x.pk);
                x.pv[0][0] = *reinterpret_cast<const uint32_t*>(par + 2 * c * 8 + 4);
                x.pv[1][0] = *reinterpret_cast<const uint32_t*>(par + (2 * c + 1) * 8 + 4);
            }
        };
        const int tk = w * 8 + g, tv = w * 8 + 2 * c;
        auto at = [&](uint8_t* t, int tok, int ch) {
            return reinterpret_cast<uint4*>(t + tok * 128 + ((ch ^ (tok & 7)) << 4));
        };
        if (c == 0) {                                  // the unused half of the lows' slots
            *at(smem + S::kLow, tk, 1) = make_uint4(0, 0, 0, 0);
            *at(smem + S::kLow + S::kTile, tk, 1) = make_uint4(0, 0, 0, 0);
        }
        Raw raw;                                       // a step ahead
        load(page_of(0), raw);
        int next = page_of(1);
        for (int i = 0; i < steps; ++i) {
            Raw ahead;
            load(next, ahead);
            next = page_of(i + 2);
            const int b = i & 1;
            if (i >= 2 && !wait(kv_free[b], (i >> 1) - 1, 256)) break;
            uint8_t* kt = smem + S::kK + b * 2 * S::kHalf;
            uint8_t* vt = smem + S::kV + b * 2 * S::kHalf;
#pragma unroll
            for (int grp = 0; grp < NG; ++grp) {
                const uint32_t s = __byte_perm(raw.pk[grp], 0, 0x1010);
#pragma unroll
                for (int x = 0; x < 2; ++x) {          // K: 8 dims of a token
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        split_product(sub_bf16x2(codes128(raw.k[2 * grp + x] >> (4 * j)), 0x43004300u), s, hi[j], lo[j]);
                    *at(kt + grp * S::kTile, tk, 2 * c + x) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *at(kt + S::kHalf + grp * S::kTile, tk, 2 * c + x) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                uint32_t e[4], o[4];                   // V: 8 dims of two tokens, n - 8
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t word = raw.v[2 * grp + j / 2] >> (8 * (j % 2));
                    const uint32_t x = sub_bf16x2(codes128(word), 0x43084308u);
                    const uint32_t y = sub_bf16x2(codes128(word >> 4), 0x43084308u);
                    e[j] = __byte_perm(x, y, 0x5410);
                    o[j] = __byte_perm(x, y, 0x7632);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t sv = __byte_perm(raw.pv[t][grp], 0, 0x1010);
                    if ((sv & 0x7F80u) == 0x7F80u) sv = 0;     // NaN: left to B
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_product(t == 0 ? e[j] : o[j], sv, hi[j], lo[j]);
                    *at(vt + 2 * grp * S::kTile, tv + t, g) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *at(vt + (2 * grp + 1) * S::kTile, tv + t, g) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            if (c == 0) {
                const uint32_t l0 = raw.pk[0] >> 16, l1 = NG == 2 ? raw.pk[NG - 1] >> 16 : 0;
                *at(smem + S::kLow + b * S::kTile, tk, 0) = make_uint4(l0 | l0 << 16, l0 | l1 << 16, l1 | l1 << 16, 0);
                const uint32_t v0 = raw.pk[NG], v1 = raw.pk[NW - 1];
                reinterpret_cast<float2*>(smem + S::kB)[b * kTcKeys + tk] =
                    make_float2(fmaf(8.f, bf16lo_to_f32(v0), bf16hi_to_f32(v0)), fmaf(8.f, bf16lo_to_f32(v1), bf16hi_to_f32(v1)));
            }
            fence_proxy_async_smem();
            mbar_arrive(smem_addr(&kv_full[b]));
            raw = ahead;
        }
    } else {
        // ---- MMA: the warp stays together, one lane issues ----
        constexpr uint32_t idesc_s = idesc_bf16_f32(kTcRows, kTcKeys, false);
        constexpr uint32_t idesc_o = idesc_bf16_f32(kTcRows, 64, true);
        // Descriptors differ in their address field (16-byte units) alone.
        const uint64_t d_qs = sdesc_sw128(sbase + S::kQs, 16, 1024), d_low = sdesc_sw128(sbase + S::kLow, 16, 1024);
        const uint64_t d_k = sdesc_sw128(sbase + S::kK, 16, 1024), d_v = sdesc_sw128(sbase + S::kV, 16, 1024);
        auto scores = [&](int b) {
            const uint32_t to = tmem + (uint32_t)(kS + b * kTcKeys);
            const uint64_t k0 = d_k + (uint32_t)(b * (2 * S::kHalf / 16));
            mma_ss(to, d_qs, d_low + (uint32_t)(b * (S::kTile / 16)), idesc_s, 0u);
#pragma unroll
            for (int hl = 0; hl < 2; ++hl)
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    mma_ts(to, tmem + (uint32_t)(kQ + kk * 8), k0 + (hl * S::kHalf + kk / 4 * S::kTile + kk % 4 * 32) / 16,
                           idesc_s, 1u);
            mma_commit(smem_addr(&s_full[b]));
        };
        auto output = [&](int i) {
            const int b = i & 1;
            const uint32_t from = tmem + (uint32_t)(kS + b * kTcKeys);
            const uint64_t v0 = d_v + (uint32_t)(b * (2 * S::kHalf / 16));
#pragma unroll
            for (int grp = 0; grp < NG; ++grp)
#pragma unroll
                for (int hl = 0; hl < 2; ++hl)
#pragma unroll
                    for (int kk = 0; kk < kTcKeys / 16; ++kk)
                        mma_ts(tmem + (uint32_t)(grp * 64), from + (uint32_t)(kk * 8),
                               v0 + ((2 * grp + hl) * S::kTile + kk * 2048) / 16, idesc_o, (i > 0 || hl > 0 || kk > 0) ? 1u : 0u);
            mma_commit(smem_addr(&o_full[b]));
            mma_commit(smem_addr(&kv_free[b]));
        };
        bool ok = wait(q_full, 0, 255);
        for (int i = 0; i <= steps && ok; ++i) {
            if (i < steps) {
                ok = wait(kv_full[i & 1], i >> 1, 255);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) scores(i & 1);
                __syncwarp();
            }
            if (i > 0) {
                ok = wait(p_full[(i - 1) & 1], (i - 1) >> 1, 259);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) output(i - 1);
                __syncwarp();
            }
        }
        if (!ok) {                                     // MMAs already issued end before the memory is released
            if (elect_one()) mma_commit(smem_addr(&drained));
            __syncwarp();
            if (lane == 0) {
                const uint64_t t0 = global_timer_ns();
                while (!mbar_try_wait(smem_addr(&drained), 0) && global_timer_ns() - t0 < 100000000ull) {
                }
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, kCols);
    if (threadIdx.x == 0 && err != 0) atomicCAS(&g_device_error, 0, err);
}

}  // namespace q4
}  // namespace lf
