// Paged split-KV decode attention over K/V pages held in 4 bits (format: q4_common.cuh).
//
// One query token per session, o = softmax(scale q k^T) v over k = n_k s_k + b_k, v = n_v s_v + b_v.
// The codes are never expanded to values.  With the scales taken out of the products,
//   q . k_t = sum over groups of  s_t (q . n_t) + b_t sum(q)
//   o       = sum over tokens of  (p_t s_t) n_t + p_t b_t,
// the matrix products run on the codes themselves.  A bf16 bit pattern below 256 stands for
// 2^-133 times the pattern: the subnormals and the first normals share their step.  So a code of bits
// 0..3 is n 2^-133 as it stands, one of bits 4..7 is 16 n 2^-133, and the two pairs of a word's low
// bytes cost one mask each, those of its high bytes one shift more; the products are exact.  The
// powers of two are balanced by 2^64 in the other operand (q, or p s, which therefore has to stay
// below 2^63: the append stores no larger scale) and removed where sums are used; the factor 16 goes
// into q, or out of every second output dim at the end.  Probabilities times scales are
// rounded to bf16; a product of the same rounded values with the constant -8 is added to o and
// b + 8 s applied with unrounded probabilities, so that the rounding (2^-9 on average) multiplies
// n - 8, centred in the range, not n.
//
// As in the bf16 decode a page's 16 tokens are the M rows of m16n8k16:
//   S^T [16 tokens x 8 columns]  = codes_k [16 x D] . q^T [D x 8]       per group, D/16 MMAs
//   O^T [D x 8 columns]         += codes_v^T [D x 16] . (p s)^T [16 x 8]  D/16 MMAs
// A warp's lane holds 16-byte vectors of codes that are its operand registers (no ldmatrix, no
// bank conflicts); a page of one KV head is one block of 18 D bytes, brought in by one bulk copy.
//
// Work:
//   own     the sessions' own pages, two at a time (a unit), in the order (session, KV head, unit),
//           are cut into equal ranges, one per resident warp, so that long and short sessions fill
//           the chip alike and a warp starts up once.  A warp works alone, with a ring of kStages
//           units whose copies run on across heads and sessions (the queries of a head come with
//           its first unit).  The columns are the GQA group's heads.
//   prefix  the pages of a shared prefix, a kernel of its own, next to which the own one starts.  Long
//           prefixes of many rows go to tiles of 128 rows on tcgen05 (decode_q4_prefix.cuh); here:
//           (chunk, KV head, group of 4 * 8/G sessions): the 8 columns of a warp are G heads of 8/G
//           sessions, and the four warps use the same staged pages, so that a prefix page is read once
//           per 32 columns.
//   few     few sessions without a prefix, e.g. one: an item (session, KV head) is a cluster of up to 8
//           CTAs, which merges its warps' partials on the chip; one launch and no workspace.
// Every other piece writes unnormalised fp32 partials (o, max, sum); a range's piece of item (session, KV
// head) is partial number range + item, which no two pieces share as both grow along the ranges.
// combine merges a row's partials, in order.
//
// Every barrier wait is bounded (site 251 in the device error word); a warp that gives up stops
// computing and lets the copies in flight land, bounded again, before it leaves.
#include "decode_common.cuh"
#include "q4_common.cuh"
#include "sm100_primitives.cuh"

#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace lf {
namespace q4 {

namespace cg = cooperative_groups;

using decode::checked_page;
using decode::kThreads;
using decode::kWarps;

// own: pages of a unit (a barrier, a softmax step, a buffer).  GP: heads of a group whose units are packed
// (4, or 1 or 2 of 64 dims), or 0.
constexpr int unit_pages(int GP) { return GP == 1 || GP == 2 ? 4 : 2; }
constexpr int kStages = 2;                     // own: units in flight per warp
constexpr int per_sm(int D) { return D == 64 ? 4 : 3; }   // own: resident CTAs of an SM (registers)
constexpr int kMinUnits = 2;                   // own: units of a range
constexpr int kRing = 16;                      // prefix: pages staged in a CTA, in two halves
constexpr int kMaxParts = 8;                   // few items: CTAs of an item, a cluster (portable size)
constexpr uint64_t kWaitNs = 2000000000ull;

struct DecodeArgs {
    const uint16_t* q;
    const uint8_t* pages;
    const int32_t *bt, *lens;
    float *own_o, *pre_o;                      // [ranges + N * Hkv][G][D]; [N][Hq][n_chunks][D]
    float2 *own_ml, *pre_ml;                   // (max, sum) of each
    int2* span;                                // [N * Hkv] first and last range of an item
    int N, Hq, Hkv, G, num_pages, max_pages;
    int n_prefix, chunk, n_chunks, groups;     // shared prefix: pages, pages a chunk, chunks, session groups
    int ranges;                                // of the own pages: one per warp
    int parts;                                 // few items: CTAs of an item (0: not few)
    uint16_t* o;
    float* lse;                                // nullable
    float qscale;                              // |scale| * log2(e) * 2^69
    uint32_t flip;                             // sign bits of a negative scale
};

__device__ __forceinline__ int held(const DecodeArgs& a, int n) {
    return n < a.N ? min(max(a.lens[n], 0), a.max_pages * kPage) : 0;
}
// Units of a session's own pages.
template <int U>
__device__ __forceinline__ int own_units(const DecodeArgs& a, int n) {
    const int own = (held(a, n) + kPage - 1) / kPage - a.n_prefix;
    return own > 0 ? (own + U - 1) / U : 0;
}

// Waits for a phase; false after kWaitNs.
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = sm100::global_timer_ns();
    while (!sm100::mbar_try_wait(bar, parity))
        if (sm100::global_timer_ns() - t0 > kWaitNs) return false;
    return true;
}
// The same for a whole warp, the answer uniform; a phase that is there costs a poll and a vote.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, sm100::mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait_full(bar, parity));
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar,
                                          uint64_t policy) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1], %2, [%3], %4;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar), "l"(policy)
        : "memory");
}

template <int NW>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&w)[NW]) {
    if constexpr (NW == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// D = A . B + C, m16n8k16, bf16 operands, fp32 accumulators.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Codes i of both halves of a word, as the bf16 pair n 2^-133 (i even) or 16 n 2^-133 (i odd).
__device__ __forceinline__ uint32_t codes(uint32_t w, int i) {
    return (i < 2 ? w : w >> 8) & (i % 2 == 0 ? 0x000F000Fu : 0x00F000F0u);
}
constexpr float kUp = 18446744073709551616.f;            // 2^64, in q and in p s
constexpr float kDown = 590295810358705651712.f;         // 2^69 = 2^133 / 2^64

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// A warp's attention state: 8 columns (query rows), of which this lane holds 2c and 2c + 1.  Scores and maxima are kept as q . k 2^-69 (q's sign carries the scale's).
template <int D, int U>
struct State {
    static constexpr int NG = Fmt<D>::NG;
    uint32_t qb[NG][4][2];                     // Q^T operand, column g: q 2^64, q 2^60
    float qsum[NG][2];                         // sums of columns 2c, 2c + 1 over each group, 2^-69
    float o[NG][4][4];                         // O^T: m-tile (16 dims) x 4; 2^-69, 2^-65 in rows g + 8
    float corr[NG][4];                         // -8 sum(bf16(p s)): the same in every m-tile
    float bias[NG][2];                         // this lane's share of sum p (b + 8 s)
    float m[2], l[2];

    // `row` is column g's query row (null: the column is unused); `flip` is 0x80008000 for a
    // negative scale.
    __device__ __forceinline__ void init(const uint16_t* row, uint32_t flip, int c) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (row != nullptr) {
                x = *reinterpret_cast<const uint4*>(row + gr * kGroup + c * 16);
                y = *reinterpret_cast<const uint4*>(row + gr * kGroup + c * 16 + 8);
            }
            const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            float part = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                qb[gr][k / 2][k % 2] = mul_bf16x2(w[k] ^ flip, k % 2 == 0 ? 0x5F805F80u : 0x5D805D80u);
                part += bf16lo_to_f32(w[k] ^ flip) + bf16hi_to_f32(w[k] ^ flip);
            }
            part += __shfl_xor_sync(0xffffffffu, part, 1);
            part += __shfl_xor_sync(0xffffffffu, part, 2);
            part *= 1.f / kDown;
            qsum[gr][0] = __shfl_sync(0xffffffffu, part, 8 * c);
            qsum[gr][1] = __shfl_sync(0xffffffffu, part, 8 * c + 4);
            bias[gr][0] = bias[gr][1] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                corr[gr][k] = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[gr][k][j] = 0.f;
            }
        }
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // Applies U staged pages, tokens tok0 .. tok0 + 16 U - 1; len: the lengths of the lane's columns.
    // kMasked: some token may be at or past a column's length.  Such tokens take no part, whatever
    // their codes and scales hold.
    template <bool kMasked>
    __device__ __forceinline__ void unit(uint32_t base, int tok0, const int (&len)[2], float qscale, int lane) {
        const int g = lane >> 2, c = lane & 3;
        float s[U][4];                     // (token g, col 2c), (g, 2c+1), (g+8, 2c), (g+8, 2c+1)
        uint32_t vp[U][2][NG];             // V params of tokens g, g + 8
#pragma unroll
        for (int pg = 0; pg < U; ++pg) {
            const uint32_t blk = base + (uint32_t)(pg * Fmt<D>::kBlockBytes);
            uint32_t pa[2 * NG], pb[2 * NG], ka[2 * NG], kb[2 * NG];
            lds<2 * NG>(blk + Fmt<D>::kParOff + g * (8 * NG), pa);
            lds<2 * NG>(blk + Fmt<D>::kParOff + (g + 8) * (8 * NG), pb);
            lds<2 * NG>(blk + g * (32 * NG) + c * (8 * NG), ka);
            lds<2 * NG>(blk + (g + 8) * (32 * NG) + c * (8 * NG), kb);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                vp[pg][0][gr] = pa[NG + gr];
                vp[pg][1][gr] = pb[NG + gr];
                float acc[4];
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t a0 = codes(ka[2 * gr + w], 2 * k), a1 = codes(kb[2 * gr + w], 2 * k);
                        const uint32_t a2 = codes(ka[2 * gr + w], 2 * k + 1), a3 = codes(kb[2 * gr + w], 2 * k + 1);
                        if (w == 0 && k == 0) {
                            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(acc, a0, a1, a2, a3, qb[gr][0][0], qb[gr][0][1], zero);
                        } else {
                            mma(acc, a0, a1, a2, a3, qb[gr][2 * w + k][0], qb[gr][2 * w + k][1], acc);
                        }
                    }
                const float sa = bf16lo_to_f32(pa[gr]), sb = bf16lo_to_f32(pb[gr]);
                const float ba = bf16hi_to_f32(pa[gr]), bb = bf16hi_to_f32(pb[gr]);
                float(&t)[4] = s[pg];
                if (gr == 0) {
                    t[0] = ba * qsum[gr][0];
                    t[1] = ba * qsum[gr][1];
                    t[2] = bb * qsum[gr][0];
                    t[3] = bb * qsum[gr][1];
                } else {
                    t[0] = fmaf(ba, qsum[gr][0], t[0]);
                    t[1] = fmaf(ba, qsum[gr][1], t[1]);
                    t[2] = fmaf(bb, qsum[gr][0], t[2]);
                    t[3] = fmaf(bb, qsum[gr][1], t[3]);
                }
                t[0] = fmaf(sa, acc[0], t[0]);
                t[1] = fmaf(sa, acc[1], t[1]);
                t[2] = fmaf(sb, acc[2], t[2]);
                t[3] = fmaf(sb, acc[3], t[3]);
            }
        }
        bool keep[U][4];
        if (kMasked) {
#pragma unroll
                for (int pg = 0; pg < U; ++pg)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        keep[pg][j] = tok0 + kPage * pg + g + 8 * (j / 2) < len[j % 2];
                        s[pg][j] = keep[pg][j] ? s[pg][j] : -INFINITY;
                    }
        }
        float x0 = fmaxf(s[0][0], s[0][2]), x1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
        for (int pg = 1; pg < U; ++pg) {
            x0 = fmaxf(x0, fmaxf(s[pg][0], s[pg][2]));
            x1 = fmaxf(x1, fmaxf(s[pg][1], s[pg][3]));
        }
        // Only lanes of the column need agree, and only when the maximum grows.
        if (__any_sync(0xffffffffu, x0 > m[0] || x1 > m[1])) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
            }
            const float n0 = fmaxf(m[0], x0), n1 = fmaxf(m[1], x1);
            const float a0 = m[0] == n0 ? 1.f : fast_exp2((m[0] - n0) * qscale);
            const float a1 = m[1] == n1 ? 1.f : fast_exp2((m[1] - n1) * qscale);
            // (a column that had met no token has sums of zero: any finite factor will do)
            const float f0 = m[0] == -INFINITY ? 0.f : a0, f1 = m[1] == -INFINITY ? 0.f : a1;
            m[0] = n0;
            m[1] = n1;
            l[0] *= f0;
            l[1] *= f1;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                bias[gr][0] *= f0;
                bias[gr][1] *= f1;
#pragma unroll
                for (int j = 0; j < 4; ++j) corr[gr][j] *= (j & 1) ? f1 : f0;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[gr][k][j] *= (j & 1) ? f1 : f0;
            }
        }
        // a column that has met no token yet keeps a maximum of -inf; its scores are all -inf
        const float r0 = (kMasked && m[0] == -INFINITY) ? 0.f : m[0] * -qscale;
        const float r1 = (kMasked && m[1] == -INFINITY) ? 0.f : m[1] * -qscale;
#pragma unroll
        for (int pg = 0; pg < U; ++pg)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = fast_exp2(fmaf(s[pg][j], qscale, (j & 1) ? r1 : r0));
                s[pg][j] = !kMasked || keep[pg][j] ? e : 0.f;
            }
#pragma unroll
        for (int pg = 0; pg < U; ++pg) {
            l[0] += s[pg][0] + s[pg][2];
            l[1] += s[pg][1] + s[pg][3];
        }
#pragma unroll
        for (int pg = 0; pg < U; ++pg) {
            const uint32_t blk = base + (uint32_t)(pg * Fmt<D>::kBlockBytes) + Fmt<D>::kVOff;
            uint32_t va[2 * NG], vb[2 * NG];   // tokens 2c, 2c + 1 and 2c + 8, 2c + 9
            lds<2 * NG>(blk + lane * (8 * NG), va);
            lds<2 * NG>(blk + 256 * NG + lane * (8 * NG), vb);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                const float sa = bf16lo_to_f32(vp[pg][0][gr]), sb = bf16lo_to_f32(vp[pg][1][gr]);
                const float ba = fmaf(8.f, sa, bf16hi_to_f32(vp[pg][0][gr]));
                const float bb = fmaf(8.f, sb, bf16hi_to_f32(vp[pg][1][gr]));
                const float ua = sa * kUp, ub = sb * kUp;
                uint32_t b0, b1;
                const float(&e)[4] = s[pg];
                float p[4] = {e[0] * ua, e[1] * ua, e[2] * ub, e[3] * ub};
                if (kMasked) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = keep[pg][j] ? p[j] : 0.f;
                    bias[gr][0] += (keep[pg][0] ? e[0] * ba : 0.f) + (keep[pg][2] ? e[2] * bb : 0.f);
                    bias[gr][1] += (keep[pg][1] ? e[1] * ba : 0.f) + (keep[pg][3] ? e[3] * bb : 0.f);
                } else {
                    bias[gr][0] = fmaf(e[0], ba, fmaf(e[2], bb, bias[gr][0]));
                    bias[gr][1] = fmaf(e[1], ba, fmaf(e[3], bb, bias[gr][1]));
                }
                b0 = movm_t(pack_bf16x2(p[0], p[1]));
                b1 = movm_t(pack_bf16x2(p[2], p[3]));
                // -8 2^-133 in rows g, -128 2^-133 in rows g + 8
                mma(corr[gr], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0, b1, corr[gr]);
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t a0 = codes(va[2 * gr + w], 2 * k), a1 = codes(va[2 * gr + w], 2 * k + 1);
                        const uint32_t a2 = codes(vb[2 * gr + w], 2 * k), a3 = codes(vb[2 * gr + w], 2 * k + 1);
                            mma(o[gr][2 * w + k], a0, a1, a2, a3, b0, b1, o[gr][2 * w + k]);
                    }
            }
        }
    }

    // The head that column g stands for, or -1.
    static __device__ __forceinline__ int head_of(int g, int G) { return g < G ? g : -1; }

    // Sums over the lanes that share a column; o then holds the whole unnormalised rows.
    __device__ __forceinline__ void finish(float) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
            l[1] += __shfl_xor_sync(0xffffffffu, l[1], off);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                bias[gr][0] += __shfl_xor_sync(0xffffffffu, bias[gr][0], off);
                bias[gr][1] += __shfl_xor_sync(0xffffffffu, bias[gr][1], off);
            }
        }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[gr][k][j] = fmaf(o[gr][k][j] + corr[gr][j], j < 2 ? kDown : kDown / 16.f, bias[gr][j & 1]);
    }
};

// The same for groups of fewer than 8 heads, a unit's pages at once: column n stands for head n % G over
// page n / G, so that the softmax's arithmetic, the same for 8 columns as for one, serves all of them.  A
// page's MMAs get the operand with the other pages' columns zero, and all add to the same accumulators.
// Columns keep their own maximum and sums; those of a head are joined at the end.
// 4 heads, 2 pages: 480 instructions a unit of 128 dims, 522 with pages in columns of their own; 64 sessions of
// 4096 .. 16384 tokens 149.5 us, 154.0.  1 or 2 heads of 64 dims, 4 pages: 96 sessions x 12 heads x 4000 tokens
// 73 us, 85; 1 to 1280 tokens 21.5 and 23.8; 64 sessions x 8 heads of 2 x 6000 53 and 61; 300 tokens 15.4
// and 14.7.  (One or two heads of 128 dims would need 4 pages of twice the size in flight: State.)
template <int D, int G>
struct Packed {
    static constexpr int U = unit_pages(G), NG = Fmt<D>::NG;
    // copies of q: one a page with the other pages' columns zero, where they fit (masked at use with 4 heads:
    // ragged 42.8 us, not 41.6)
    static constexpr int QM = U == 2 ? U : 1;
    uint32_t qb[QM][NG][4][2];                 // Q^T operand, column g: q 2^64, q 2^60
    float qsum[NG][2];
    float o[NG][4][4];
    float corr[NG][4];
    float bias[NG][2];
    float m[2], l[2];

    static __device__ __forceinline__ int head_of(int g, int) { return g < U * G ? g % G : -1; }

    __device__ __forceinline__ void init(const uint16_t* row, uint32_t flip, int c) {
        State<D, 1> one;
        one.init(row, flip, c);
        const int page = (threadIdx.x & 31) / 4 / G;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int q = 0; q < QM; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j) qb[q][gr][k][j] = QM == 1 || page == q ? one.qb[gr][k][j] : 0u;
                corr[gr][k] = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[gr][k][j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                qsum[gr][j] = one.qsum[gr][j];
                bias[gr][j] = 0.f;
            }
        }
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    template <bool kMasked>
    __device__ __forceinline__ void unit(uint32_t base, int tok0, const int (&len)[2], float qscale, int lane) {
        using F = Fmt<D>;
        const int g = lane >> 2, c = lane & 3;
        constexpr int kAcc = 2;                // chains of MMAs a group (one: ragged 41.6 us, two 41.2)
        float acc[kAcc][NG][4];
#pragma unroll
        for (int p = 0; p < U; ++p) {
            const uint32_t blk = base + (uint32_t)(p * F::kBlockBytes);
            const uint32_t sel = QM > 1 || g / G == p ? 0xFFFFFFFFu : 0u;
            uint32_t ka[2 * NG], kb[2 * NG];
            lds<2 * NG>(blk + g * (32 * NG) + c * (8 * NG), ka);
            lds<2 * NG>(blk + (g + 8) * (32 * NG) + c * (8 * NG), kb);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float(&d)[4] = acc[p * kAcc / U][gr];
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t a0 = codes(ka[2 * gr + w], 2 * k), a1 = codes(kb[2 * gr + w], 2 * k);
                        const uint32_t a2 = codes(ka[2 * gr + w], 2 * k + 1), a3 = codes(kb[2 * gr + w], 2 * k + 1);
                        const uint32_t(&q)[2] = qb[QM > 1 ? p : 0][gr][2 * w + k];
                        if (p % (U / kAcc) == 0 && w == 0 && k == 0) {
                            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(d, a0, a1, a2, a3, q[0] & sel, q[1] & sel, zero);
                        } else {
                            mma(d, a0, a1, a2, a3, q[0] & sel, q[1] & sel, d);
                        }
                    }
            }
        }
        // This lane's columns 2c, 2c + 1 and the pages they stand for (past the last one: any page, masked).
        const int page[2] = {(2 * c / G) % U, ((2 * c + 1) / G) % U};
        const bool live = 2 * c < U * G;
        float s[4];                            // (token g, col 2c), (g, 2c+1), (g+8, 2c), (g+8, 2c+1)
        float vs[4][NG], vb[4][NG];
        bool keep[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (G > 1 && j % 2 == 1) continue;           // the same page: below
            uint32_t par[2 * NG];
            lds<2 * NG>(base + (uint32_t)(page[j % 2] * F::kBlockBytes + F::kParOff + (g + 8 * (j / 2)) * (8 * NG)), par);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                const float ks = bf16lo_to_f32(par[gr]), kl = bf16hi_to_f32(par[gr]);
                vs[j][gr] = bf16lo_to_f32(par[NG + gr]);
                vb[j][gr] = fmaf(8.f, vs[j][gr], bf16hi_to_f32(par[NG + gr]));
#pragma unroll
                for (int i = 0; i < (G > 1 ? 2 : 1); ++i) {
                    float x = acc[0][gr][j + i];
                    if (kAcc > 1) x += acc[kAcc - 1][gr][j + i];
                    const float y = kl * qsum[gr][(j + i) % 2];
                    s[j + i] = gr == 0 ? fmaf(ks, x, y) : fmaf(ks, x, fmaf(kl, qsum[gr][(j + i) % 2], s[j + i]));
                }
                if (G > 1) {
                    vs[j + 1][gr] = vs[j][gr];
                    vb[j + 1][gr] = vb[j][gr];
                }
            }
        }
        constexpr bool kSome = kMasked || U * G < 8;     // some columns or tokens do not count
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            keep[j] = live && (!kMasked || tok0 + kPage * page[j % 2] + g + 8 * (j / 2) < len[0]);
            if (kSome) s[j] = keep[j] ? s[j] : -INFINITY;
        }
        float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
        if (__any_sync(0xffffffffu, x0 > m[0] || x1 > m[1])) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
            }
            const float n0 = fmaxf(m[0], x0), n1 = fmaxf(m[1], x1);
            const float f0 = m[0] == -INFINITY ? 0.f : (m[0] == n0 ? 1.f : fast_exp2((m[0] - n0) * qscale));
            const float f1 = m[1] == -INFINITY ? 0.f : (m[1] == n1 ? 1.f : fast_exp2((m[1] - n1) * qscale));
            m[0] = n0;
            m[1] = n1;
            l[0] *= f0;
            l[1] *= f1;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                bias[gr][0] *= f0;
                bias[gr][1] *= f1;
#pragma unroll
                for (int j = 0; j < 4; ++j) corr[gr][j] *= (j & 1) ? f1 : f0;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[gr][k][j] *= (j & 1) ? f1 : f0;
            }
        }
        const float r0 = m[0] == -INFINITY ? 0.f : m[0] * -qscale, r1 = m[1] == -INFINITY ? 0.f : m[1] * -qscale;
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            e[j] = fast_exp2(fmaf(s[j], qscale, (j & 1) ? r1 : r0));
            if (kSome) e[j] = keep[j] ? e[j] : 0.f;
            l[j & 1] += e[j];
        }
        uint32_t b0[NG], b1[NG];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            float p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {      // what a masked token's scales hold does not count
                float& bs = bias[gr][j & 1];
                bs = kSome ? bs + (keep[j] ? e[j] * vb[j][gr] : 0.f) : fmaf(e[j], vb[j][gr], bs);
                p[j] = e[j] * (vs[j][gr] * kUp);
                if (kSome) p[j] = keep[j] ? p[j] : 0.f;
            }
            b0[gr] = movm_t(pack_bf16x2(p[0], p[1]));
            b1[gr] = movm_t(pack_bf16x2(p[2], p[3]));
            mma(corr[gr], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0[gr], b1[gr], corr[gr]);
        }
#pragma unroll
        for (int q = 0; q < U; ++q) {
            const uint32_t blk = base + (uint32_t)(q * F::kBlockBytes) + F::kVOff + lane * (8 * NG);
            const uint32_t sel = g / G == q ? 0xFFFFFFFFu : 0u;
            uint32_t va[2 * NG], vc[2 * NG];   // tokens 2c, 2c + 1 and 2c + 8, 2c + 9
            lds<2 * NG>(blk, va);
            lds<2 * NG>(blk + 256 * NG, vc);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        mma(o[gr][2 * w + k], codes(va[2 * gr + w], 2 * k), codes(va[2 * gr + w], 2 * k + 1),
                            codes(vc[2 * gr + w], 2 * k), codes(vc[2 * gr + w], 2 * k + 1), b0[gr] & sel, b1[gr] & sel,
                            o[gr][2 * w + k]);
        }
    }

    // Sums over lanes and over the columns of a head; columns 0 .. G - 1 then hold the rows.
    __device__ __forceinline__ void finish(float qscale) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[j] += __shfl_xor_sync(0xffffffffu, l[j], off);
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) bias[gr][j] += __shfl_xor_sync(0xffffffffu, bias[gr][j], off);
            }
        }
        constexpr int kFirst = G == 4 ? 2 : 1; // lanes of a head's columns: c and those kFirst, 2 kFirst, ... away
        float M[2] = {m[0], m[1]};
        if (G == 1) M[0] = M[1] = fmaxf(M[0], M[1]);
#pragma unroll
        for (int off = kFirst; off < 4; off <<= 1)
#pragma unroll
            for (int j = 0; j < 2; ++j) M[j] = fmaxf(M[j], __shfl_xor_sync(0xffffffffu, M[j], off));
        float w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            // (a column that has met no token has sums of zero, or of NaN: any finite weight will do)
            w[j] = m[j] == M[j] ? 1.f : (m[j] == -INFINITY ? 0.f : fast_exp2((m[j] - M[j]) * qscale));
            m[j] = M[j];
        }
        auto join = [&](float x0, float x1, float& y0, float& y1) {
            x0 *= w[0];
            x1 *= w[1];
            if (G == 1) x0 += x1;
#pragma unroll
            for (int off = kFirst; off < 4; off <<= 1) {
                x0 += __shfl_xor_sync(0xffffffffu, x0, off);
                if (G > 1) x1 += __shfl_xor_sync(0xffffffffu, x1, off);
            }
            y0 = x0;
            y1 = x1;
        };
        join(l[0], l[1], l[0], l[1]);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[gr][k][j] = fmaf(o[gr][k][j] + corr[gr][j], j < 2 ? kDown : kDown / 16.f, bias[gr][j & 1]);
                join(o[gr][k][0], o[gr][k][1], o[gr][k][0], o[gr][k][1]);
                join(o[gr][k][2], o[gr][k][3], o[gr][k][2], o[gr][k][3]);
            }
    }
};
template <int D, int GP> struct StateOf { typedef Packed<D, GP> T; };
template <int D> struct StateOf<D, 0> { typedef State<D, 2> T; };

// Dim of accumulator row g of m-tile k of group gr (row g + 8 is the next dim).
__device__ __forceinline__ int out_dim(int gr, int k, int g) { return gr * kGroup + 8 * g + 2 * k; }

// -- own pages ----------------------------------------------------------------------------------------
template <int D, int GP>
struct OwnSmem {
    static constexpr int kUnitBytes = unit_pages(GP) * Fmt<D>::kBlockBytes;
    static constexpr int kQ = 8 * D * 2;                   // queries of a KV head, at most 8 rows
    static constexpr int kWarp = kStages * kUnitBytes + 2 * kQ;
    static constexpr int kBytes = kWarps * kWarp + 128;
    // few items: the warps' partials, [warp][row][D] fp32 and [warp][row] (max, sum)
    static constexpr int kPart = kWarps * kWarp, kPartMl = kPart + kWarps * 8 * D * 4;
    static constexpr int kFewBytes = kPartMl + kWarps * 8 * 8 + 128;
};

// Sum over the CTA's threads (every thread gets it).
__device__ __forceinline__ long cta_sum(long v, long* buf) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    long r = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) r += buf[w];
    __syncthreads();
    return r;
}

// A run of units [j, j1) of (session n, KV head h), and how many units follow it in the range.
struct Segment {
    int n, h, j, j1, u, L;
    long left;
    // Moves on to the next segment; false at the range's end.
    template <int U>
    __device__ __forceinline__ bool next(const DecodeArgs& a) {
        if (left <= 0) return false;
        if (++h == a.Hkv) {
            h = 0;
            do { u = own_units<U>(a, ++n); } while (u == 0 && n < a.N);
            if (u == 0) return false;                            // (not met: units are left)
            L = held(a, n);
        }
        j = 0;
        j1 = (int)min((long)u, left);
        left -= j1;
        return true;
    }
};

__device__ __forceinline__ uint8_t* align128(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 127) & ~uintptr_t(127));
}
// A warp's barriers, one a unit in flight.
__device__ __forceinline__ uint32_t init_ring(uint64_t* bars, int lane) {
    const uint32_t bar = sm100::smem_addr(bars);
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) sm100::mbar_init(bar + 8 * i, 1);
        sm100::fence_barrier_init();
    }
    return bar;
}

// A warp's segments, from `seg` on: copies, products, partials.  kFew: to the CTA's shared memory (part_o
// [warp][8 rows][D]), else to the range's slots.  (`a` by value: by reference the ragged case takes 42.1
// us, not 41.2.)
template <int D, int GP, bool kFew>
__device__ __forceinline__ void run_segments(const DecodeArgs a, Segment seg, int range, uint8_t* mem, uint32_t bar,
                                             float* part_o, float2* part_ml) {
    using F = Fmt<D>;
    constexpr int U = unit_pages(GP), UB = OwnSmem<D, GP>::kUnitBytes;
    typedef typename StateOf<D, GP>::T St;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint8_t* qbuf = mem + kStages * UB;
    const uint32_t ring = sm100::smem_addr(mem), qring = ring + kStages * UB;
    // What it copies: a segment that runs ahead.  Page ids of 32 / U units at a time, one page per
    // lane (lane U i + p: page p of the i-th).
    Segment pre = seg;
    bool more = true, fresh = true;                          // fresh: the segment's first unit
    int ids = 0, ids_at = 32 / U;
    uint32_t issued = 0, used = 0, q_in = 0;
    const uint64_t policy = sm100::l2_evict_first_policy();  // read once
    auto issue = [&]() {                                     // warp-uniform: one unit, if any is left
        if (more && pre.j >= pre.j1) {
            more = pre.template next<U>(a);
            fresh = true;
            ids_at = 32 / U;
        }
        if (!more) return;
        if (ids_at == 32 / U) {
            ids_at = 0;
            const int p = a.n_prefix + (pre.j + lane / U) * U + lane % U;
            ids = p < (pre.L + kPage - 1) / kPage ? checked_page(a.bt[(size_t)pre.n * a.max_pages + p], a.num_pages) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, ids, ids_at * U + lane % U);
        const int n_pages = __popc(__ballot_sync(0xffffffffu, lane < U && page >= 0));
        const int st = issued % kStages;
        const uint32_t q_bytes = a.G * D * 2;
        if (lane == 0)
            sm100::mbar_arrive_expect_tx(bar + 8 * st, n_pages * F::kBlockBytes + (fresh ? q_bytes : 0));
        __syncwarp();
        if (lane < U && page >= 0)
            bulk_load(ring + (uint32_t)(st * UB + lane * F::kBlockBytes),
                      a.pages + ((size_t)page * a.Hkv + pre.h) * F::kBlockBytes, F::kBlockBytes, bar + 8 * st, policy);
        if (fresh && lane == U)
            bulk_load(qring + (q_in & 1) * OwnSmem<D, GP>::kQ, a.q + ((size_t)pre.n * a.Hq + pre.h * a.G) * D, q_bytes,
                      bar + 8 * st, policy);
        q_in += fresh;
        fresh = false;
        ++issued;
        ++ids_at;
        ++pre.j;
    };
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kStages; ++k) issue();
    uint32_t q_out = 0;
    bool failed = false;
    do {
        const int item = seg.n * a.Hkv + seg.h, L = seg.L;
        const int len[2] = {L, L};
        St st;
        for (int j = seg.j; j < seg.j1; ++j) {
            const int sl = used % kStages;
            if (!warp_wait(bar + 8 * sl, (used / kStages) & 1)) {
                if (lane == 0) {
                    atomicCAS(&g_device_error, 0, 251);      // let the copies in flight land
                    for (uint32_t k = used; k < issued; ++k) wait_full(bar + 8 * (k % kStages), (k / kStages) & 1);
                }
                failed = true;
                break;
            }
            if (j == seg.j) {
                const uint16_t* rows = reinterpret_cast<const uint16_t*>(qbuf + (q_out & 1) * OwnSmem<D, GP>::kQ);
                const int head = St::head_of(g, a.G);
                st.init(head >= 0 ? rows + head * D : nullptr, a.flip, c);
                ++q_out;
            }
            const uint32_t blk = ring + (uint32_t)(sl * UB);
            const int tok0 = (a.n_prefix + j * U) * kPage;
            if (tok0 + U * kPage <= L) st.template unit<false>(blk, tok0, len, a.qscale, lane);
            else st.template unit<true>(blk, tok0, len, a.qscale, lane);
            __syncwarp();                                    // every lane has read the buffer
            ++used;
            issue();
        }
        if (failed) break;
        st.finish(a.qscale);
        // Columns 2c and 2c + 1 are heads of the group; lane g holds 2 dims of each m-tile.
        const size_t slot = kFew ? (size_t)warp * 8 : (size_t)(range + item) * a.G;
        float* out_o = kFew ? part_o : a.own_o;
        float2* out_ml = kFew ? part_ml : a.own_ml;
#pragma unroll
        for (int col = 0; col < 2; ++col) {
            if (2 * c + col >= a.G) continue;
            float* dst = out_o + (slot + 2 * c + col) * D;
#pragma unroll
            for (int gr = 0; gr < F::NG; ++gr)
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                    *reinterpret_cast<float4*>(dst + out_dim(gr, k, g)) =
                        make_float4(st.o[gr][k][col], st.o[gr][k][2 + col],
                                    st.o[gr][k + 1][col], st.o[gr][k + 1][2 + col]);
            if (g == 0) out_ml[slot + 2 * c + col] = make_float2(st.m[col], st.l[col]);
        }
        if (!kFew && lane == 0) {
            if (seg.j == 0) a.span[item].x = range;
            if (seg.j1 == seg.u) a.span[item].y = range;
        }
    } while (seg.template next<U>(a));
}

template <int V> struct Vec;
template <> struct Vec<2> { typedef float2 T; };
template <> struct Vec<4> { typedef float4 T; };

// Weighted sum of `count` partials of a row, this lane's V dims: x(t) and ml(t) are loaded all at once.
template <int V, int kMax, class X, class ML>
__device__ __forceinline__ float2 merge_row(int count, float qscale, X x, ML ml, float (&acc)[V]) {
    typedef typename Vec<V>::T VT;
    VT v[kMax];
    float2 e[kMax];
#pragma unroll
    for (int t = 0; t < kMax; ++t) {
        e[t] = t < count ? *ml(t) : make_float2(-INFINITY, 0.f);
        if (t < count) v[t] = *reinterpret_cast<const VT*>(x(t));
    }
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int t = 0; t < kMax; ++t) M = fmaxf(M, e[t].x);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int t = 0; t < kMax; ++t)
        if (e[t].y != 0.f) {                                     // (0: no token, and nothing was written)
            const float w = e[t].x == M ? 1.f : fast_exp2((e[t].x - M) * qscale);
            const float* f = reinterpret_cast<const float*>(&v[t]);
            l = fmaf(w, e[t].y, l);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = fmaf(w, f[i], acc[i]);
        }
    return make_float2(M, l);
}

// The final rows of a cluster's item: over a CTA's warps, then over the CTAs through distributed shared
// memory, a row each.
template <int D>
__device__ void merge_few(const DecodeArgs& a, float* part_o, float2* part_ml) {
    constexpr int V = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cg::cluster_group cluster = cg::this_cluster();
    float acc[V];
    __syncthreads();
    for (int r = warp; r < a.G; r += kWarps) {
        const float2 e = merge_row<V, kWarps>(kWarps, a.qscale, [&](int w) { return part_o + (w * 8 + r) * D + V * lane; },
                                              [&](int w) { return part_ml + w * 8 + r; }, acc);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) part_o[r * D + V * lane + i] = acc[i];
        if (lane == 0) part_ml[r] = e;
    }
    cluster.sync();
    const int item = blockIdx.x / a.parts, n = item / a.Hkv;
    for (int r = (int)cluster.block_rank() + warp * a.parts; r < a.G; r += kWarps * a.parts) {
        const float2 e = merge_row<V, kMaxParts>(
            a.parts, a.qscale, [&](int t) { return cluster.map_shared_rank(part_o + r * D + V * lane, t); },
            [&](int t) { return cluster.map_shared_rank(part_ml + r, t); }, acc);
        const size_t row = (size_t)n * a.Hq + item % a.Hkv * a.G + r;
        const float inv = e.y != 0.f ? 1.f / e.y : 0.f;
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.o + row * D) + (V / 2) * lane;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) dst[i] = pack_bf16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
        if (a.lse != nullptr && lane == 0)
            a.lse[row] = e.y != 0.f ? (e.x * a.qscale + log2f(e.y)) * kLn2 : -INFINITY;
    }
    cluster.sync();                                              // others may still read this CTA's shared memory
}

template <int D, int GP>
__global__ void __launch_bounds__(kThreads, per_sm(D)) own_kernel(const DecodeArgs a) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kWarps * kStages];
    __shared__ long buf[kWarps];
    __shared__ long s_before[kWarps];          // units of one head before session s_n[w]
    __shared__ int s_n[kWarps];
    // Inputs are there after grid_wait(), or, behind the prefix kernel, from the start (it waited before
    // it let this one begin); combine may read the lengths as soon as it is released.
    if (a.n_chunks == 0) grid_wait();
    grid_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* mem = align128(smem_raw) + warp * OwnSmem<D, GP>::kWarp;
    const uint32_t bar = init_ring(bars + warp * kStages, lane);
    // Units of a CTA's width of sessions, summed up to each: the first such chunk serves the total and,
    // in most batches, the search.
    long excl = 0, chunk = 0;                                    // units before this thread's session; of the chunk
    int u = 0;
    auto scan = [&](int n0) {
        u = n0 + threadIdx.x < a.N ? own_units<unit_pages(GP)>(a, n0 + threadIdx.x) : 0;
        long incl = u;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) buf[warp] = incl;
        __syncthreads();
        excl = incl - u;
        chunk = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) excl += buf[w];
            chunk += buf[w];
        }
        __syncthreads();
    };
    scan(0);
    long total = chunk;
    if (a.N > kThreads) {
        long mine = 0;
        for (int n = kThreads + threadIdx.x; n < a.N; n += kThreads) mine += own_units<unit_pages(GP)>(a, n);
        total += cta_sum(mine, buf);
    }
    total *= a.Hkv;
    const long share = max((total + a.ranges - 1) / a.ranges, (long)kMinUnits);
    const int range = blockIdx.x * kWarps + warp;
    const long begin = range * share, cta_begin = (long)blockIdx.x * kWarps * share;
    const long cta_last = min(cta_begin + (kWarps - 1) * share, total - 1);
    if (cta_begin < total) {                                     // the sessions where the CTA's ranges start
        long before = 0;
        for (int n0 = 0;;) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const long at = cta_begin + w * share, from = before + excl;
                if (at >= from * a.Hkv && at < (from + u) * a.Hkv) {
                    s_before[w] = from;
                    s_n[w] = n0 + threadIdx.x;
                }
            }
            before += chunk;
            n0 += kThreads;
            if (n0 >= a.N || before * a.Hkv > cta_last) break;
            scan(n0);
        }
        __syncthreads();
    }
    if (begin < total) {
        Segment seg;
        seg.n = s_n[warp];
        seg.u = own_units<unit_pages(GP)>(a, seg.n);
        seg.L = held(a, seg.n);
        const long in = begin - s_before[warp] * a.Hkv, len = min(share, total - begin);
        seg.h = (int)(in / seg.u);
        seg.j = (int)(in % seg.u);
        seg.j1 = (int)min((long)seg.u, seg.j + len);
        seg.left = len - (seg.j1 - seg.j);
        run_segments<D, GP, false>(a, seg, range, mem, bar, nullptr, nullptr);
    }
    if (a.n_chunks > 0) grid_wait();                             // the prefix kernel's partials are there too
}

// Few items without a prefix.  An item is a cluster's: its units are cut over the cluster's warps, whose
// partials are merged on the chip, so that the call is one launch.
template <int D, int GP>
__global__ void __launch_bounds__(kThreads, per_sm(D)) few_kernel(const DecodeArgs a) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[kWarps * kStages];
    grid_wait();
    grid_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = align128(smem_raw);
    float* part_o = reinterpret_cast<float*>(smem + OwnSmem<D, GP>::kPart);
    float2* part_ml = reinterpret_cast<float2*>(smem + OwnSmem<D, GP>::kPartMl);
    if (lane < 8) part_ml[warp * 8 + lane] = make_float2(-INFINITY, 0.f);
    const uint32_t bar = init_ring(bars + warp * kStages, lane);
    const int item = blockIdx.x / a.parts, w = blockIdx.x % a.parts * kWarps + warp;
    Segment seg;
    seg.n = item / a.Hkv;
    seg.h = item % a.Hkv;
    seg.u = own_units<unit_pages(GP)>(a, seg.n);
    seg.L = held(a, seg.n);
    const int share = (seg.u + a.parts * kWarps - 1) / (a.parts * kWarps);
    seg.j = w * share;
    seg.j1 = min(seg.u, seg.j + share);
    seg.left = 0;
    if (seg.j < seg.j1) run_segments<D, GP, true>(a, seg, 0, smem + warp * OwnSmem<D, GP>::kWarp, bar, part_o, part_ml);
    merge_few<D>(a, part_o, part_ml);
}

// -- shared prefix --------------------------------------------------------------------------------------
template <int D>
struct PrefixSmem {
    static constexpr int kBytes = kRing * Fmt<D>::kBlockBytes + 128;
};

// One chunk of the prefix for the sessions of four warps (8 columns each) of one KV head.  The staged pages are a ring of two halves, refilled half by half after a CTA barrier.
template <int D>
__global__ void __launch_bounds__(kThreads, 4) prefix_kernel(const DecodeArgs a) {
    using F = Fmt<D>;
    constexpr int kHalf = kRing / 2;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    __shared__ __align__(8) uint64_t bars[kRing];
    grid_wait();
    grid_release();                                              // the own pages need nothing from here
    const int chunk = blockIdx.x % a.n_chunks, h = blockIdx.x / a.n_chunks % a.Hkv;
    const int group = blockIdx.x / a.n_chunks / a.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int spb = 8 / a.G;                                     // sessions of a block
    const int first = group * kWarps * spb;
    const int p_begin = chunk * a.chunk, p_end = min(p_begin + a.chunk, a.n_prefix);
    // The page ids come from the group's longest session, whose row holds every page that any
    // session here needs; pages past its length are not read.
    int best = -1, lead = first;
    for (int i = lane; i < kWarps * spb; i += 32) {
        const int L = held(a, first + i);
        if (L > best) { best = L; lead = first + i; }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const int ob = __shfl_xor_sync(0xffffffffu, best, off), ol = __shfl_xor_sync(0xffffffffu, lead, off);
        if (ob > best || (ob == best && ol < lead)) { best = ob; lead = ol; }
    }
    const int pages = min(p_end, (best + kPage - 1) / kPage) - p_begin;
    if (pages <= 0) return;                                      // combine reads no slot of this chunk
    const int32_t* row = a.bt + (size_t)lead * a.max_pages + p_begin;
    const uint32_t ring = sm100::smem_addr(smem), bar = sm100::smem_addr(bars);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) sm100::mbar_init(bar + 8 * i, 1);
        sm100::fence_barrier_init();
    }
    __syncthreads();
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    auto issue_half = [&](int k0) {                              // pages k0 .. k0 + kHalf - 1, one a lane of warp 0
        const int k = k0 + lane;
        if (warp == 0 && lane < kHalf && k < pages) {
            const int sl = k % kRing, page = checked_page(row[k], a.num_pages);
            sm100::mbar_arrive_expect_tx(bar + 8 * sl, F::kBlockBytes);
            bulk_load(ring + (uint32_t)(sl * F::kBlockBytes),
                      a.pages + ((size_t)page * a.Hkv + h) * F::kBlockBytes, F::kBlockBytes, bar + 8 * sl, policy);
        }
    };
    issue_half(0);
    issue_half(kHalf);
    State<D, 1> st;
    const int base = first + warp * spb, n_g = base + g / a.G;
    const int len[2] = {held(a, base + (2 * c) / a.G), held(a, base + (2 * c + 1) / a.G)};
    int lmin = min(len[0], len[1]);
    st.init(n_g < a.N ? a.q + ((size_t)n_g * a.Hq + h * a.G + g % a.G) * D : nullptr, a.flip, c);
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) lmin = min(lmin, __shfl_xor_sync(0xffffffffu, lmin, off));
    bool failed = false;
    for (int k0 = 0; k0 < pages; k0 += kHalf) {
        for (int k = k0; k < min(k0 + kHalf, pages); ++k) {
            const int sl = k % kRing;
            if (!failed && !warp_wait(bar + 8 * sl, (uint32_t)((k / kRing) & 1))) {
                if (lane == 0) atomicCAS(&g_device_error, 0, 251);
                failed = true;
            }
            if (failed) continue;
            const uint32_t blk = ring + (uint32_t)(sl * F::kBlockBytes);
            const int tok0 = (p_begin + k) * kPage;
            if (tok0 + kPage <= lmin) st.template unit<false>(blk, tok0, len, a.qscale, lane);
            else st.template unit<true>(blk, tok0, len, a.qscale, lane);
        }
        if (__syncthreads_or(failed)) {                          // every warp is done with this half
            const int k = k0 + lane;                             // copies may still be landing
            if (warp == 0 && lane < kRing && k < pages) wait_full(bar + 8 * (k % kRing), (uint32_t)((k / kRing) & 1));
            break;
        }
        issue_half(k0 + kRing);
    }
    st.finish(a.qscale);
    // rows of columns 2c and 2c + 1 go straight to their slots
#pragma unroll
    for (int col = 0; col < 2; ++col) {
        const int j = 2 * c + col, n = base + j / a.G;
        if (n >= a.N) continue;
        const size_t slot = ((size_t)n * a.Hq + h * a.G + j % a.G) * a.n_chunks + chunk;
#pragma unroll
        for (int gr = 0; gr < F::NG; ++gr)
#pragma unroll
            for (int k = 0; k < 4; k += 2)
                *reinterpret_cast<float4*>(a.pre_o + slot * D + out_dim(gr, k, g)) =
                    make_float4(st.o[gr][k][col], st.o[gr][k][2 + col], st.o[gr][k + 1][col], st.o[gr][k + 1][2 + col]);
        if (g == 0) a.pre_ml[slot] = make_float2(st.m[col], st.l[col]);
    }
}

}  // namespace q4
}  // namespace lf

#include "decode_q4_prefix.cuh"

namespace lf {
namespace q4 {

// Merges the partials of a row (session, query head), the prefix chunks first, by their maxima.  A row
// without tokens gives zeros and an lse of -inf.  R warps a row: 1, or kRowWarps where a row has many
// partials (they take 32 of them in turn).
constexpr int kRowWarps = 8, kManyPartials = 32;
template <int D, int R>
__global__ void __launch_bounds__(R == 1 ? kThreads : 32 * R)
combine_kernel(const DecodeArgs a) {
    constexpr int kRows = R == 1 ? kWarps : 1;             // rows of a CTA
    const int lane = threadIdx.x & 31, part = R == 1 ? 0 : threadIdx.x >> 5;
    const long row = (long)blockIdx.x * kRows + (R == 1 ? threadIdx.x >> 5 : 0);
    if (row >= (long)a.N * a.Hq) return;
    const int n = (int)(row / a.Hq), hq = (int)(row % a.Hq), item = n * a.Hkv + hq / a.G;
    const int npages = (held(a, n) + kPage - 1) / kPage;
    const int chunks = a.n_prefix > 0 ? (min(npages, a.n_prefix) + a.chunk - 1) / a.chunk : 0;
    grid_wait();                                              // the partials are written
    int2 span = npages > a.n_prefix ? a.span[item] : make_int2(0, -1);
    span.x = max(0, min(span.x, a.ranges - 1));               // (a range that gave up leaves any bits there)
    span.y = max(span.x - 1, min(span.y, a.ranges - 1));
    const int total = chunks + span.y - span.x + 1;
    const long own0 = (long)(span.x + item) * a.G + hq % a.G, pre0 = row * a.n_chunks;
    auto ml = [&](int j) { return j < chunks ? a.pre_ml[pre0 + j] : a.own_ml[own0 + (long)(j - chunks) * a.G]; };
    constexpr int V = D / 32;                              // dims of a lane
    auto vec = [&](int j) {
        return (j < chunks ? a.pre_o + (pre0 + j) * D : a.own_o + (own0 + (long)(j - chunks) * a.G) * D) + V * lane;
    };
    typedef typename Vec<V>::T VT;
    // Vectors come in batches of kBatch at once, the first while the weights are formed.
    constexpr int kBatch = 8;
    VT x[kBatch];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int t = 0; t < kBatch; ++t)
            if (t0 + t < total) x[t] = *reinterpret_cast<const VT*>(vec(t0 + t));
    };
    fetch(32 * part);
    float2 e = make_float2(-INFINITY, 0.f);
    if (lane < total) e = ml(lane);
    float M = e.x;
    for (int j = lane + 32; j < total; j += 32) M = fmaxf(M, ml(j).x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float acc[V], l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
    float w = 0.f;
    for (int j0 = R == 1 ? 0 : 32 * part; j0 < total; j0 += kBatch) {
        if (j0 % 32 == 0) {                                // weights of 32 slots, one a lane
            if (j0 > 0) e = j0 + lane < total ? ml(j0 + lane) : make_float2(-INFINITY, 0.f);
            w = e.x == -INFINITY ? 0.f : fast_exp2((e.x - ref) * a.qscale);
            l = fmaf(w, e.y, l);
        }
        if (j0 > (R == 1 ? 0 : 32 * part)) fetch(j0);
#pragma unroll
        for (int t = 0; t < kBatch; ++t) {
            const float wt = __shfl_sync(0xffffffffu, w, (j0 + t) % 32);
            const float* f = reinterpret_cast<const float*>(&x[t]);
            if (j0 + t < total)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = fmaf(wt, f[i], acc[i]);
        }
        if constexpr (R > 1) j0 += j0 % 32 == 32 - kBatch ? 32 * (R - 1) : 0;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if constexpr (R > 1) {                                 // the warps' sums, in order
        __shared__ float s_acc[R][D], s_l[R];
#pragma unroll
        for (int i = 0; i < V; ++i) s_acc[part][V * lane + i] = acc[i];
        if (lane == 0) s_l[part] = l;
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int p = 1; p < R; ++p) {
            l += s_l[p];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += s_acc[p][V * lane + i];
        }
    }
    const float inv = total > 0 && l != 0.f ? 1.f / l : 0.f;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.o + row * D) + (V / 2) * lane;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dst[i] = pack_bf16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    if (a.lse != nullptr && lane == 0) a.lse[row] = l != 0.f ? (ref * a.qscale + log2f(l)) * kLn2 : -INFINITY;
}

// -- sizes ------------------------------------------------------------------------------------------
inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// Whether the prefix goes to tiles of 128 rows on tcgen05.  Both forms' times grow with rows x pages x
// heads, the tiles' at less than half the rate but from 4 us more (barriers, tensor memory, more code to
// fetch); they meet at about 2^25 row-pages x KV heads x dims.  Rows 64 x heads 8 of 128: 1024 pages 45
// against 47 us, 512 pages 36 : 33; 128 rows: 512 pages 39 : 45, 256 pages 33 : 31; 256 rows: 512 pages
// 47 : 74, 256 pages 37 : 45, 128 pages 31 : 31, 64 pages 29 : 25; 400 rows: 128 pages 36 : 41, 64 pages
// 31 : 29.  64 dims: 512 rows x 4 heads: 512 pages 37 : 51, 256 pages 29 : 33, 128 pages 25 : 25.
// (Decode times, a few own pages included.)  Up to 64 rows a tile is too empty.
inline bool prefix_on_tc(int N, int G, int Hkv, int D, int n_prefix) {
    return (long)N * G > 64 && (long)N * G * n_prefix * Hkv * D >= (1L << 25);
}

// Pages of a prefix chunk: as many chunks as keep every CTA resident at once (kTcPerSm an SM, of whole
// steps; or four an SM, of 8 pages at least).
inline int prefix_chunk(int N, int G, int Hkv, int D, int n_prefix, int sms) {
    if (n_prefix <= 0) return 1;
    if (prefix_on_tc(N, G, Hkv, D, n_prefix)) {
        const long tiles = ceil_div((long)N * G, kTcRows), steps = ceil_div(n_prefix, kTcPages);
        const long chunks = std::max(1L, std::min((long)kTcPerSm * sms / (tiles * Hkv), steps));
        return ceil_div(steps, chunks) * kTcPages;
    }
    const long groups = ceil_div((long)N * G, 8 * kWarps);
    const long chunks = std::max(1L, std::min(4L * sms / (groups * Hkv), n_prefix / 8L));
    return ceil_div(n_prefix, chunks);
}

// CTAs of an item when there are few items without a prefix (0: not few): 8, 4 or 2 that are all resident
// at once.  A cluster is alone with its item's length, so the table may allow 16 pages a warp at most.
// Of equal lengths, 8 heads of 128: 1 session of 777 tokens 6.5 against 10.2 us (two launches, partials
// through memory), 8000: 13.0 : 14.3, 16000: 20.1 : 17.1; 12 sessions of 777: 9.9 : 13.0, 4000: 19.8 :
// 24.6; 24 of 777: 13.3 : 16.4.
inline int few_parts(int N, int Hkv, int D, int n_prefix, int max_pages, int sms) {
    if (n_prefix > 0) return 0;
    int parts = kMaxParts;
    while (parts > 1 && (long)N * Hkv * parts > (long)per_sm(D) * sms) parts /= 2;
    return parts > 1 && max_pages <= 64 * parts ? parts : 0;
}

// Sizes of the workspace's parts, in their order.
struct Sizes {
    size_t own, pre, items;                    // partials of the ranges, of the prefix; spans
    int chunk, n_chunks, ranges, parts;
    size_t bytes(int D) const { return (own + pre) * (D * sizeof(float) + sizeof(float2)) + items * sizeof(int2); }
};
inline Sizes sizes(int N, int Hq, int Hkv, int D, int n_prefix, int max_pages, int sms) {
    Sizes s;
    s.parts = few_parts(N, Hkv, D, n_prefix, max_pages, sms);
    s.ranges = n_prefix < max_pages && s.parts == 0 ? per_sm(D) * sms * kWarps : 0;
    s.items = s.parts == 0 ? (size_t)N * Hkv : 0;
    s.own = s.ranges > 0 ? (s.ranges + s.items) * (Hq / Hkv) : 0;
    s.chunk = prefix_chunk(N, Hq / Hkv, Hkv, D, n_prefix, sms);
    s.n_chunks = ceil_div(n_prefix, s.chunk);
    s.pre = (size_t)N * Hq * s.n_chunks;
    return s;
}

static int sm_count(int* out) {
    int dev = 0;
    LF_CHECK_CUDA(cudaGetDevice(&dev));
    LF_CHECK_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return LF_OK;
}

// The own pages' kernel runs beside the prefix kernel, so both ask for the same split of the L1, which an SM
// changes only when it is idle (96 sessions x 12 heads of 64 on 64 pages: 18.4 us, 24.6 otherwise; beside
// the tiles, which leave no room for it, it makes no difference to ask).
inline int prepare(void (*kernel)(DecodeArgs), int bytes) {
    LF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    LF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    return LF_OK;
}

template <int D, int GP>
static int launch_own(const DecodeArgs& a, cudaStream_t st) {
    static PerContextOnce once;
    const int rc = once.run([] {
        const int e = prepare(own_kernel<D, GP>, OwnSmem<D, GP>::kBytes);
        return e != LF_OK ? e : prepare(few_kernel<D, GP>, OwnSmem<D, GP>::kFewBytes);
    });
    if (rc != LF_OK) return rc;
    return a.parts > 0
               ? launch_early_clusters("q4 decode", few_kernel<D, GP>, a.parts, dim3((unsigned)(a.N * a.Hkv * a.parts)),
                                       dim3(kThreads), OwnSmem<D, GP>::kFewBytes, st, a)
               : launch_early("q4 decode", own_kernel<D, GP>, dim3(a.ranges / kWarps), dim3(kThreads),
                              OwnSmem<D, GP>::kBytes, st, a);
}
template <int D>
static int launch_own_of(const DecodeArgs& a, cudaStream_t st) {
    if constexpr (D == 64) {
        if (a.G == 1) return launch_own<64, 1>(a, st);
        if (a.G == 2) return launch_own<64, 2>(a, st);
    }
    if (a.G == 4) return launch_own<D, 4>(a, st);
    return launch_own<D, 0>(a, st);
}

template <int D>
static int launch(const DecodeArgs& a, cudaStream_t st) {
    if (a.parts > 0) return launch_own_of<D>(a, st);
    static PerContextOnce once;
    int rc = once.run([] {
        LF_CHECK_CUDA(cudaFuncSetAttribute(prefix_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           TcSmem<D>::kBytes));
        return prepare(prefix_kernel<D>, PrefixSmem<D>::kBytes);
    });
    if (rc != LF_OK) return rc;
    const long shared = (long)a.n_chunks * a.Hkv * a.groups, rows = (long)a.N * a.Hq;
    LF_CHECK_ARG(shared <= 2147483647L, "q4 decode: grid limits exceeded");
    if (shared > 0) {
        rc = prefix_on_tc(a.N, a.G, a.Hkv, D, a.n_prefix)
                 ? launch_early("q4 decode prefix", prefix_tc_kernel<D>, dim3((unsigned)shared), dim3(kTcThreads),
                                TcSmem<D>::kBytes, st, a)
                 : launch_early("q4 decode prefix", prefix_kernel<D>, dim3((unsigned)shared), dim3(kThreads),
                                PrefixSmem<D>::kBytes, st, a);
        if (rc != LF_OK) return rc;
    }
    if (a.ranges > 0) {
        rc = launch_own_of<D>(a, st);
        if (rc != LF_OK) return rc;
    }
    // A row's partials, at most: the prefix chunks and an equal share of the ranges.
    const long most = a.n_chunks + std::min((long)a.ranges / (a.N * a.Hkv), (long)a.max_pages / (2 * kMinUnits)) + 1;
    return most > kManyPartials
               ? launch_early("q4 decode combine", combine_kernel<D, kRowWarps>, dim3((unsigned)rows), dim3(32 * kRowWarps),
                              0, st, a)
               : launch_early("q4 decode combine", combine_kernel<D, 1>, dim3((unsigned)ceil_div(rows, kWarps)),
                              dim3(kThreads), 0, st, a);
}

}  // namespace q4
}  // namespace lf

using namespace lf;

extern "C" int lf_q4_decode_workspace_size(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                           int max_pages, int num_prefix_pages, int sm_count, size_t* bytes) {
    LF_CHECK_ARG(bytes != nullptr, "q4 decode: bytes is null");
    LF_CHECK_ARG(num_seqs >= 0 && num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 &&
                     head_dim > 0 && max_pages > 0 && num_prefix_pages >= 0 && num_prefix_pages <= max_pages,
                 "q4 decode: bad workspace arguments");
    if (sm_count <= 0) {
        const int rc = q4::sm_count(&sm_count);
        if (rc != LF_OK) return rc;
    }
    *bytes = q4::sizes(num_seqs, num_q_heads, num_kv_heads, head_dim, num_prefix_pages, max_pages, sm_count).bytes(head_dim);
    clear_error();
    return LF_OK;
}

extern "C" int lf_q4_decode_fwd(const lf_bf16* q, const void* pages, const int32_t* block_table,
                                const int32_t* seq_lens, int num_prefix_pages, lf_bf16* o, float* lse,
                                void* workspace, size_t workspace_bytes, int num_seqs, int num_q_heads,
                                int num_kv_heads, int head_dim, int num_pages, int max_pages, float scale,
                                int sm_count, void* stream) {
    LF_CHECK_ARG(num_seqs >= 0, "q4 decode: negative sizes");
    if (num_seqs == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(q && pages && block_table && seq_lens && o, "q4 decode: null pointer argument");
    LF_CHECK_ARG(aligned16(q) && aligned16(pages) && aligned16(o) && aligned16(workspace),
                 "q4 decode: q, pages, o and workspace must be 16-byte aligned");
    LF_CHECK_ARG(head_dim == 128 || head_dim == 64, "q4 decode: head_dim must be 64 or 128 (got %d)", head_dim);
    LF_CHECK_ARG(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
                 "q4 decode: need Hq a multiple of Hkv");
    const int G = num_q_heads / num_kv_heads;
    LF_CHECK_ARG(G == 1 || G == 2 || G == 4 || G == 8, "q4 decode: Hq/Hkv must be 1, 2, 4 or 8 (got %d)", G);
    LF_CHECK_ARG(num_pages > 0 && max_pages > 0 && max_pages <= (1 << 26),
                 "q4 decode: num_pages and max_pages must be > 0 (at most 2^26 pages a session)");
    LF_CHECK_ARG((long)num_seqs * num_q_heads <= (1L << 30), "q4 decode: too many sessions");
    LF_CHECK_ARG(num_prefix_pages >= 0 && num_prefix_pages <= max_pages,
                 "q4 decode: num_prefix_pages out of range");
    if (sm_count <= 0) {
        const int rc = q4::sm_count(&sm_count);
        if (rc != LF_OK) return rc;
    }
    const q4::Sizes z = q4::sizes(num_seqs, num_q_heads, num_kv_heads, head_dim, num_prefix_pages, max_pages, sm_count);
    LF_CHECK_ARG(workspace != nullptr || z.bytes(head_dim) == 0, "q4 decode: null pointer argument");
    LF_CHECK_ARG(workspace_bytes >= z.bytes(head_dim), "q4 decode: workspace too small (%zu < %zu bytes)",
                 workspace_bytes, z.bytes(head_dim));
    q4::DecodeArgs a{};
    a.q = q;
    a.pages = static_cast<const uint8_t*>(pages);
    a.bt = block_table;
    a.lens = seq_lens;
    a.own_o = static_cast<float*>(workspace);
    a.pre_o = a.own_o + z.own * head_dim;
    a.own_ml = reinterpret_cast<float2*>(a.pre_o + z.pre * head_dim);
    a.pre_ml = a.own_ml + z.own;
    a.span = reinterpret_cast<int2*>(a.pre_ml + z.pre);
    a.N = num_seqs;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.G = G;
    a.num_pages = num_pages;
    a.max_pages = max_pages;
    a.n_prefix = num_prefix_pages;
    a.chunk = z.chunk;
    a.n_chunks = z.n_chunks;
    a.groups = q4::prefix_on_tc(num_seqs, G, num_kv_heads, head_dim, num_prefix_pages)
                   ? q4::ceil_div((long)num_seqs * G, q4::kTcRows)
                   : q4::ceil_div(num_seqs, q4::kWarps * (8 / G));
    a.ranges = z.ranges;
    a.parts = z.parts;
    a.o = o;
    a.lse = lse;
    a.qscale = fabsf(scale) * kLog2e * q4::kDown;
    a.flip = scale < 0.f ? 0x80008000u : 0u;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return head_dim == 128 ? q4::launch<128>(a, st) : q4::launch<64>(a, st);
}
