// Paged split-KV decode attention over K/V pages held in 4 bits (format: q4_common.cuh).
//
// One query token per session, o = softmax(scale q k^T) v over k = n_k s_k + b_k, v = n_v s_v + b_v.
// The codes are never expanded to values.  With the scales taken out of the products,
//   q . k_t = sum over groups of  s_t (q . n_t) + b_t sum(q)
//   o       = sum over tokens of  (p_t s_t) n_t + p_t b_t,
// the matrix products run on the codes themselves: (word >> 4 i) & 0x000F000F, or-ed with 0x4300
// twice, is a pair of bf16 operands 128 + n, exact, one shift and one logic instruction a pair.  The
// 128 goes into the bias of the scores (b - 128 s), and is removed from the output with a product
// by the constant -136 on the same bf16 probabilities: what the rounding of p s to bf16 multiplies
// is then n - 8, centred in the range, and b + 8 s is applied with unrounded fp32 probabilities.
//
// As in the bf16 decode a page's 16 tokens are the M rows of m16n8k16:
//   S^T [16 tokens x 8 columns]  = codes_k [16 x D] . q^T [D x 8]       per group, D/16 MMAs
//   O^T [D x 8 columns]         += codes_v^T [D x 16] . (p s)^T [16 x 8]  D/16 MMAs
// A warp's lane holds 16-byte vectors of codes that are its operand registers (no ldmatrix, no
// bank conflicts); a page of one KV head is one block of 18 D bytes, brought in by one bulk copy.
//
// Work items (CTAs of four warps):
//   own     (split, KV head, session): the columns are the GQA group's heads; the warps take the
//           split's pages round-robin, each with its own ring of kOwnStages pages.
//   prefix  (chunk, KV head, group of 4 * 8/G sessions): the pages of a shared prefix; the 8
//           columns of a warp are G heads of 8/G sessions, and the four warps use the same staged
//           pages for different sessions, so that a prefix page is read once per 32 columns.
// Every item writes unnormalised fp32 partials (o, max, sum) to its slots; combine merges a row's
// slots in slot order.
//
// Every barrier wait is bounded (site 221 in the device error word); a warp that gives up stops
// computing and lets the copies in flight land, bounded again, before it leaves.
#include "decode_common.cuh"
#include "q4_common.cuh"
#include "sm100_primitives.cuh"

#include <math.h>

namespace lf {
namespace q4 {

using decode::checked_page;
using decode::kThreads;
using decode::kWarps;

constexpr int kStages = 4;                     // pages in flight per warp
constexpr int kSlots = kWarps * kStages;       // page buffers of a CTA
constexpr uint64_t kWaitNs = 2000000000ull;

struct DecodeArgs {
    const uint16_t* q;
    const uint8_t* pages;
    const int32_t *bt, *lens;
    float* part_o;
    float2* part_ml;
    int N, Hq, Hkv, G, num_pages, max_pages;
    int n_prefix, chunk, n_chunks, groups;     // shared prefix: pages, pages a chunk, chunks, session groups
    int pps, max_split, n_slots;
    float qscale;                              // scale * log2(e)
};

__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = sm100::global_timer_ns();
    while (!sm100::mbar_try_wait(bar, parity))
        if (sm100::global_timer_ns() - t0 > kWaitNs) return false;
    return true;
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

// D += A . B, m16n8k16, bf16 operands, fp32 accumulators.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes 4 i .. 4 i + 3 of both halves of a word as the bf16 pair 128 + n.
__device__ __forceinline__ uint32_t codes(uint32_t w, int i) {
    uint32_t r;                                // (w & mask) | bits: one instruction
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w >> (4 * i)), "n"(0x000F000F), "r"(0x43004300u));
    return r;
}

// A warp's attention state: 8 columns (query rows), of which this lane holds 2c and 2c + 1.
template <int D>
struct State {
    static constexpr int NG = Fmt<D>::NG;
    uint32_t qb[NG][4][2];                     // Q^T operand, column g
    float qsum[NG][2];                         // sums of columns 2c, 2c + 1 over each group
    float o[NG][4][4];                         // O^T: m-tile (16 dims) x 4
    float corr[NG][4];                         // -136 sum(bf16(p s)): rows are equal
    float bias[NG][2];                         // this lane's share of sum p (b + 8 s)
    float m0, m1, l0, l1;

    // `row` is column g's query row (null: the column is unused).
    __device__ __forceinline__ void init(const uint16_t* row, int c) {
        float part[NG];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            uint4 a = make_uint4(0, 0, 0, 0), b = a;
            if (row != nullptr) {
                a = *reinterpret_cast<const uint4*>(row + gr * kGroup + c * 16);
                b = *reinterpret_cast<const uint4*>(row + gr * kGroup + c * 16 + 8);
            }
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            part[gr] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qb[gr][k][0] = w[2 * k];
                qb[gr][k][1] = w[2 * k + 1];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) part[gr] += bf16lo_to_f32(w[k]) + bf16hi_to_f32(w[k]);
            part[gr] += __shfl_xor_sync(0xffffffffu, part[gr], 1);
            part[gr] += __shfl_xor_sync(0xffffffffu, part[gr], 2);
            qsum[gr][0] = __shfl_sync(0xffffffffu, part[gr], 8 * c);
            qsum[gr][1] = __shfl_sync(0xffffffffu, part[gr], 8 * c + 4);
            bias[gr][0] = bias[gr][1] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                corr[gr][k] = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[gr][k][j] = 0.f;
            }
        }
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
    }

    // Applies one staged page whose first token is `tok0`; L0, L1 are the lengths of columns 2c and
    // 2c + 1.  kMasked: some token of the page may be at or past a column's length.  Such tokens
    // take no part, whatever their codes and scales hold.
    template <bool kMasked>
    __device__ __forceinline__ void page(uint32_t blk, int tok0, int L0, int L1, float qscale, int lane) {
        const int g = lane >> 2, c = lane & 3;
        uint32_t pa[2 * NG], pb[2 * NG];       // params of tokens g, g + 8: K groups, V groups
        lds<2 * NG>(blk + Fmt<D>::kParOff + g * (8 * NG), pa);
        lds<2 * NG>(blk + Fmt<D>::kParOff + (g + 8) * (8 * NG), pb);
        float s[4] = {0.f, 0.f, 0.f, 0.f};     // (token g, col 2c), (g, 2c+1), (g+8, 2c), (g+8, 2c+1)
        {
            uint32_t ka[2 * NG], kb[2 * NG];
            lds<2 * NG>(blk + g * (32 * NG) + c * (8 * NG), ka);
            lds<2 * NG>(blk + (g + 8) * (32 * NG) + c * (8 * NG), kb);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        mma(acc, codes(ka[2 * gr + w], 2 * k), codes(kb[2 * gr + w], 2 * k),
                            codes(ka[2 * gr + w], 2 * k + 1), codes(kb[2 * gr + w], 2 * k + 1),
                            qb[gr][2 * w + k][0], qb[gr][2 * w + k][1]);
                const float sa = bf16lo_to_f32(pa[gr]), sb = bf16lo_to_f32(pb[gr]);
                const float ba = fmaf(-128.f, sa, bf16hi_to_f32(pa[gr]));
                const float bb = fmaf(-128.f, sb, bf16hi_to_f32(pb[gr]));
                s[0] = fmaf(sa, acc[0], fmaf(ba, qsum[gr][0], s[0]));
                s[1] = fmaf(sa, acc[1], fmaf(ba, qsum[gr][1], s[1]));
                s[2] = fmaf(sb, acc[2], fmaf(bb, qsum[gr][0], s[2]));
                s[3] = fmaf(sb, acc[3], fmaf(bb, qsum[gr][1], s[3]));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] *= qscale;
        bool keep[4] = {true, true, true, true};
        if (kMasked) {
            keep[0] = tok0 + g < L0;
            keep[1] = tok0 + g < L1;
            keep[2] = tok0 + g + 8 < L0;
            keep[3] = tok0 + g + 8 < L1;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = keep[j] ? s[j] : -INFINITY;
        }
        float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
        }
        if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float a0 = m0 == n0 ? 1.f : fast_exp2(m0 - n0), a1 = m1 == n1 ? 1.f : fast_exp2(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= a0;
            l1 *= a1;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                bias[gr][0] *= a0;
                bias[gr][1] *= a1;
#pragma unroll
                for (int j = 0; j < 4; ++j) corr[gr][j] *= (j & 1) ? a1 : a0;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[gr][k][j] *= (j & 1) ? a1 : a0;
            }
        }
        // a column that has met no token yet keeps a maximum of -inf; its scores are all -inf
        const float r0 = (kMasked && m0 == -INFINITY) ? 0.f : m0, r1 = (kMasked && m1 == -INFINITY) ? 0.f : m1;
        float e[4] = {fast_exp2(s[0] - r0), fast_exp2(s[1] - r1), fast_exp2(s[2] - r0), fast_exp2(s[3] - r1)};
        l0 += e[0] + e[2];
        l1 += e[1] + e[3];
        uint32_t va[2 * NG], vb[2 * NG];       // tokens 2c, 2c + 1 and 2c + 8, 2c + 9
        lds<2 * NG>(blk + Fmt<D>::kVOff + lane * (8 * NG), va);
        lds<2 * NG>(blk + Fmt<D>::kVOff + 256 * NG + lane * (8 * NG), vb);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            const float sa = bf16lo_to_f32(pa[NG + gr]), sb = bf16lo_to_f32(pb[NG + gr]);
            const float ba = fmaf(8.f, sa, bf16hi_to_f32(pa[NG + gr]));
            const float bb = fmaf(8.f, sb, bf16hi_to_f32(pb[NG + gr]));
            float p[4] = {e[0] * sa, e[1] * sa, e[2] * sb, e[3] * sb};
            float t0 = e[0] * ba, t1 = e[1] * ba, t2 = e[2] * bb, t3 = e[3] * bb;
            if (kMasked) {
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = keep[j] ? p[j] : 0.f;
                t0 = keep[0] ? t0 : 0.f;
                t1 = keep[1] ? t1 : 0.f;
                t2 = keep[2] ? t2 : 0.f;
                t3 = keep[3] ? t3 : 0.f;
            }
            bias[gr][0] += t0 + t2;
            bias[gr][1] += t1 + t3;
            const uint32_t b0 = movm_t(pack_bf16x2(p[0], p[1])), b1 = movm_t(pack_bf16x2(p[2], p[3]));
            mma(corr[gr], 0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u, b0, b1);   // bf16 -136
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    mma(o[gr][2 * w + k], codes(va[2 * gr + w], 2 * k), codes(va[2 * gr + w], 2 * k + 1),
                        codes(vb[2 * gr + w], 2 * k), codes(vb[2 * gr + w], 2 * k + 1), b0, b1);
        }
    }

    // Sums over the lanes that share a column; o then holds the whole unnormalised rows.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, off);
            l1 += __shfl_xor_sync(0xffffffffu, l1, off);
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
                for (int j = 0; j < 4; ++j) o[gr][k][j] += corr[gr][j & 1] + bias[gr][j & 1];
    }
};

// Dim of accumulator row g of m-tile k of group gr (row g + 8 is the next dim).
__device__ __forceinline__ int out_dim(int gr, int k, int g) { return gr * kGroup + 8 * g + 2 * k; }

template <int D>
struct Smem {
    static constexpr int kRing = kSlots * Fmt<D>::kBlockBytes;
    static constexpr int kMerge = kWarps * 8 * (D + 2) * 4;
    static constexpr int kBytes = (kRing > kMerge ? kRing : kMerge) + 128;
};

// Own pages of one session: one split of one KV head.
template <int D>
__device__ __forceinline__ void own_item(const DecodeArgs& a, uint8_t* smem, uint64_t* bars, int split,
                                         int h, int n) {
    using F = Fmt<D>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int L = min(max(a.lens[n], 0), a.max_pages * kPage);
    const int npages = (L + kPage - 1) / kPage;
    const int p_begin = a.n_prefix + split * a.pps;
    if (p_begin >= npages) return;
    const int n_local = min(a.pps, npages - p_begin);
    const int mine = n_local > warp ? (n_local - warp + kWarps - 1) / kWarps : 0;
    const int32_t* row = a.bt + (size_t)n * a.max_pages;
    const uint32_t ring = sm100::smem_addr(smem) + (uint32_t)(warp * kStages * F::kBlockBytes);
    const uint32_t bar = sm100::smem_addr(bars + warp * kStages);
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) sm100::mbar_init(bar + 8 * i, 1);
        sm100::fence_barrier_init();
    }
    __syncwarp();
    const uint64_t policy = sm100::l2_evict_first_policy();      // read once
    int ids = 0, batch = -1;
    auto issue = [&](int k) {                                    // warp-uniform
        if (k >= mine) return;
        if ((k >> 5) != batch) {                                 // ids of 32 pages, one per lane
            batch = k >> 5;
            const int j = warp + kWarps * ((batch << 5) + lane);
            ids = j < n_local ? checked_page(row[p_begin + j], a.num_pages) : 0;
        }
        const int page = __shfl_sync(0xffffffffu, ids, k & 31);
        if (lane == 0) {
            const int st = k % kStages;
            sm100::mbar_arrive_expect_tx(bar + 8 * st, F::kBlockBytes);
            bulk_load(ring + (uint32_t)(st * F::kBlockBytes),
                      a.pages + ((size_t)page * a.Hkv + h) * F::kBlockBytes, F::kBlockBytes, bar + 8 * st, policy);
        }
    };
#pragma unroll
    for (int k = 0; k < kStages; ++k) issue(k);
    State<D> st;
    st.init(g < a.G ? a.q + ((size_t)n * a.Hq + h * a.G + g) * D : nullptr, c);
    bool failed = false;
    int done = 0;
    for (int k = 0; k < mine; ++k) {
        const int sl = k % kStages;
        if (!__all_sync(0xffffffffu, wait_full(bar + 8 * sl, (uint32_t)((k / kStages) & 1)))) {
            if (lane == 0) atomicCAS(&g_device_error, 0, 221);
            failed = true;
            break;
        }
        done = k + 1;
        const uint32_t blk = ring + (uint32_t)(sl * F::kBlockBytes);
        const int tok0 = (p_begin + warp + kWarps * k) * kPage;
        if (tok0 + kPage <= L) st.template page<false>(blk, tok0, L, L, a.qscale, lane);
        else st.template page<true>(blk, tok0, L, L, a.qscale, lane);
        __syncwarp();                                            // every lane has read the buffer
        issue(k + kStages);
    }
    if (failed && lane == 0)                                     // let the copies in flight land
        for (int k = done + 1; k < min(mine, done + kStages); ++k)
            wait_full(bar + 8 * (k % kStages), (uint32_t)((k / kStages) & 1));
    st.finish();

    __syncthreads();                                             // the rings are idle: merge in them
    float* sm_m = reinterpret_cast<float*>(smem);                // [kWarps][8]
    float* sm_l = sm_m + kWarps * 8;
    float* sm_o = sm_l + kWarps * 8;                             // [kWarps][8][D]
    if (g == 0) {
        sm_m[warp * 8 + 2 * c] = st.m0;
        sm_m[warp * 8 + 2 * c + 1] = st.m1;
        sm_l[warp * 8 + 2 * c] = st.l0;
        sm_l[warp * 8 + 2 * c + 1] = st.l1;
    }
#pragma unroll
    for (int gr = 0; gr < F::NG; ++gr)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float* r0 = sm_o + (size_t)(warp * 8 + 2 * c) * D + out_dim(gr, k, g);
            *reinterpret_cast<float2*>(r0) = make_float2(st.o[gr][k][0], st.o[gr][k][2]);
            *reinterpret_cast<float2*>(r0 + D) = make_float2(st.o[gr][k][1], st.o[gr][k][3]);
        }
    __syncthreads();
    for (int idx = threadIdx.x; idx < a.G * D; idx += kThreads) {
        const int hd = idx / D, d = idx % D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w * 8 + hd]);
        float acc = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = sm_m[w * 8 + hd];
            if (mw == -INFINITY && sm_l[w * 8 + hd] == 0.f) continue;   // a warp without pages
            const float sc = fast_exp2(mw - M);
            acc = fmaf(sc, sm_o[(size_t)(w * 8 + hd) * D + d], acc);
            l = fmaf(sc, sm_l[w * 8 + hd], l);
        }
        const size_t slot = ((size_t)n * a.Hq + h * a.G + hd) * a.n_slots + a.n_chunks + split;
        a.part_o[slot * D + d] = acc;
        if (d == 0) a.part_ml[slot] = make_float2(M, l);
    }
}

// One chunk of the shared prefix for 4 * 8/G sessions of one KV head.  The page buffers are one ring
// of two halves of kSlots / 2 pages, refilled half by half after a CTA barrier.
template <int D>
__device__ __forceinline__ void prefix_item(const DecodeArgs& a, uint8_t* smem, uint64_t* bars, int chunk,
                                            int h, int group) {
    using F = Fmt<D>;
    constexpr int kHalf = kSlots / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int spw = 8 / a.G;                                     // sessions of a warp
    const int first = group * kWarps * spw;
    const int p_begin = chunk * a.chunk, p_end = min(p_begin + a.chunk, a.n_prefix);
    auto held = [&](int n) { return n < a.N ? min(max(a.lens[n], 0), a.max_pages * kPage) : 0; };
    // The page ids come from the group's longest session, whose row holds every page that any
    // session here needs; pages past its length are not read.
    int best = -1, lead = first;
    for (int i = 0; i < kWarps * spw; ++i) {
        const int L = held(first + i);
        if (L > best) { best = L; lead = first + i; }
    }
    const int pages = min(p_end, (best + kPage - 1) / kPage) - p_begin;
    if (pages <= 0) return;                                      // combine reads no slot of this chunk
    const int32_t* row = a.bt + (size_t)lead * a.max_pages + p_begin;
    const uint32_t ring = sm100::smem_addr(smem), bar = sm100::smem_addr(bars);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) sm100::mbar_init(bar + 8 * i, 1);
        sm100::fence_barrier_init();
    }
    __syncthreads();
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    auto issue_half = [&](int k0) {                              // pages k0 .. k0 + kHalf - 1, warp 0
        const int k = k0 + lane;
        if (warp == 0 && lane < kHalf && k < pages) {
            const int page = checked_page(row[k], a.num_pages);
            const int sl = k % kSlots;
            sm100::mbar_arrive_expect_tx(bar + 8 * sl, F::kBlockBytes);
            bulk_load(ring + (uint32_t)(sl * F::kBlockBytes),
                      a.pages + ((size_t)page * a.Hkv + h) * F::kBlockBytes, F::kBlockBytes, bar + 8 * sl, policy);
        }
    };
    issue_half(0);
    issue_half(kHalf);
    const int base = first + warp * spw;                         // this warp's sessions
    const int n_g = base + g / a.G, L0 = held(base + (2 * c) / a.G), L1 = held(base + (2 * c + 1) / a.G);
    State<D> st;
    st.init(n_g < a.N ? a.q + ((size_t)n_g * a.Hq + h * a.G + g % a.G) * D : nullptr, c);
    int lmin = min(L0, L1);
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) lmin = min(lmin, __shfl_xor_sync(0xffffffffu, lmin, off));
    bool failed = false;
    for (int k0 = 0; k0 < pages; k0 += kHalf) {
        for (int k = k0; k < min(k0 + kHalf, pages); ++k) {
            const int sl = k % kSlots;
            if (!failed && !__all_sync(0xffffffffu, wait_full(bar + 8 * sl, (uint32_t)((k / kSlots) & 1)))) {
                if (lane == 0) atomicCAS(&g_device_error, 0, 221);
                failed = true;
            }
            if (failed) continue;
            const uint32_t blk = ring + (uint32_t)(sl * F::kBlockBytes);
            const int tok0 = (p_begin + k) * kPage;
            if (tok0 + kPage <= lmin) st.template page<false>(blk, tok0, L0, L1, a.qscale, lane);
            else st.template page<true>(blk, tok0, L0, L1, a.qscale, lane);
        }
        if (__syncthreads_or(failed)) {                          // every warp is done with this half
            const int k = k0 + lane;                             // copies may still be landing
            if (warp == 0 && lane < kSlots && k < pages) wait_full(bar + 8 * (k % kSlots), (uint32_t)((k / kSlots) & 1));
            break;
        }
        issue_half(k0 + kSlots);
    }
    st.finish();
    // rows of columns 2c and 2c + 1 go straight to their slots
#pragma unroll
    for (int col = 0; col < 2; ++col) {
        const int j = 2 * c + col, n = base + j / a.G;
        if (n >= a.N) continue;
        const size_t slot = ((size_t)n * a.Hq + h * a.G + j % a.G) * a.n_slots + chunk;
#pragma unroll
        for (int gr = 0; gr < F::NG; ++gr)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float2*>(a.part_o + slot * D + out_dim(gr, k, g)) =
                    make_float2(st.o[gr][k][col], st.o[gr][k][2 + col]);
        if (g == 0) a.part_ml[slot] = col ? make_float2(st.m1, st.l1) : make_float2(st.m0, st.l0);
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads) decode_kernel(const DecodeArgs a) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    __shared__ __align__(8) uint64_t bars[kSlots];
    long item = blockIdx.x;
    const long n_pre = (long)a.n_chunks * a.Hkv * a.groups;
    if (item < n_pre) {
        const int chunk = (int)(item % a.n_chunks);
        item /= a.n_chunks;
        prefix_item<D>(a, smem, bars, chunk, (int)(item % a.Hkv), (int)(item / a.Hkv));
        return;
    }
    item -= n_pre;
    const int split = (int)(item % a.max_split);
    item /= a.max_split;
    own_item<D>(a, smem, bars, split, (int)(item % a.Hkv), (int)(item / a.Hkv));
}

// One warp per (session, query head): merges the row's partials, the prefix chunks first, by their
// maxima.  A row without tokens gives zeros and an lse of -inf.
template <int D>
__global__ void __launch_bounds__(kThreads)
combine_kernel(const DecodeArgs a, uint16_t* __restrict__ o, float* __restrict__ lse) {
    const int lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= (long)a.N * a.Hq) return;
    const int n = (int)(row / a.Hq);
    const int L = min(max(a.lens[n], 0), a.max_pages * kPage);
    const int npages = (L + kPage - 1) / kPage;
    const int chunks = a.n_prefix > 0 ? (min(npages, a.n_prefix) + a.chunk - 1) / a.chunk : 0;
    const int splits = npages > a.n_prefix ? (npages - a.n_prefix + a.pps - 1) / a.pps : 0;
    const int total = chunks + splits;
    const float2* ml = a.part_ml + row * a.n_slots;
    const float* po = a.part_o + row * (long)a.n_slots * D;
    auto slot = [&](int j) { return j < chunks ? j : a.n_chunks + (j - chunks); };
    float M = -INFINITY;
    for (int j = lane; j < total; j += 32) M = fmaxf(M, ml[slot(j)].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    constexpr int V = D / 32;                              // dims of a lane
    float acc[V], l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    const float ref = M == -INFINITY ? 0.f : M;
    for (int j0 = 0; j0 < total; j0 += 32) {
        float w = 0.f;
        if (j0 + lane < total) {
            const float2 e = ml[slot(j0 + lane)];
            w = fast_exp2(e.x - ref);
            l = fmaf(w, e.y, l);
        }
        const int end = min(32, total - j0);
#pragma unroll 4
        for (int t = 0; t < end; ++t) {
            const float wt = __shfl_sync(0xffffffffu, w, t);
            const float* src = po + (long)slot(j0 + t) * D + V * lane;
            if constexpr (V == 4) {
                const float4 x = *reinterpret_cast<const float4*>(src);
                acc[0] = fmaf(wt, x.x, acc[0]);
                acc[1] = fmaf(wt, x.y, acc[1]);
                acc[2] = fmaf(wt, x.z, acc[2]);
                acc[3] = fmaf(wt, x.w, acc[3]);
            } else {
                const float2 x = *reinterpret_cast<const float2*>(src);
                acc[0] = fmaf(wt, x.x, acc[0]);
                acc[1] = fmaf(wt, x.y, acc[1]);
            }
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const float inv = total > 0 && l != 0.f ? 1.f / l : 0.f;
    uint32_t* dst = reinterpret_cast<uint32_t*>(o + row * D) + (V / 2) * lane;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) dst[i] = pack_bf16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    if (lse != nullptr && lane == 0) lse[row] = l != 0.f ? (M + log2f(l)) * kLn2 : -INFINITY;
}

// -- sizes ------------------------------------------------------------------------------------------
inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// Pages of a prefix chunk: halved from the whole prefix down to 16 while the items stay under about
// four per SM.
inline int prefix_chunk(int N, int G, int Hkv, int n_prefix, int sms) {
    const long groups = ceil_div((long)N * G, 8 * kWarps);
    int c = n_prefix;
    while (c > 16 && groups * Hkv * ceil_div(n_prefix, c) < 4L * sms) c = (c + 1) / 2;
    return c > 0 ? c : 1;
}

inline int own_splits(int max_pages, int n_prefix, int pps) { return ceil_div(max_pages - n_prefix, pps); }

constexpr int kMinChunk = 16;
inline size_t slots_bound(int max_pages, int n_prefix, int pps) {
    return (size_t)own_splits(max_pages, n_prefix, pps) + (size_t)ceil_div(n_prefix, kMinChunk / 2);
}

static int sm_count(int* out) {
    int dev = 0;
    LF_CHECK_CUDA(cudaGetDevice(&dev));
    LF_CHECK_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    return LF_OK;
}

template <int D>
static int launch(const DecodeArgs& a, uint16_t* o, float* lse, cudaStream_t st) {
    static PerContextOnce once;
    const int rc = once.run([] {
        LF_CHECK_CUDA(cudaFuncSetAttribute(decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           Smem<D>::kBytes));
        return LF_OK;
    });
    if (rc != LF_OK) return rc;
    const long items = (long)a.n_chunks * a.Hkv * a.groups + (long)a.max_split * a.Hkv * a.N;
    LF_CHECK_ARG(items <= 2147483647L, "q4 decode: grid limits exceeded");
    if (items > 0) {
        decode_kernel<D><<<(unsigned)items, kThreads, Smem<D>::kBytes, st>>>(a);
        const int e = launch_status("q4 decode");
        if (e != LF_OK) return e;
    }
    const long rows = (long)a.N * a.Hq;
    combine_kernel<D><<<(unsigned)ceil_div(rows, kWarps), kThreads, 0, st>>>(a, o, lse);
    return launch_status("q4 decode combine");
}

}  // namespace q4
}  // namespace lf

using namespace lf;

extern "C" int lf_q4_decode_default_split(int num_seqs, int num_kv_heads, int max_pages,
                                          int num_prefix_pages, int sm_count, int* pages_per_split) {
    LF_CHECK_ARG(pages_per_split != nullptr, "q4 decode split: out pointer is null");
    LF_CHECK_ARG(num_seqs >= 0 && num_kv_heads > 0 && max_pages > 0 && num_prefix_pages >= 0 &&
                     num_prefix_pages <= max_pages,
                 "q4 decode split: bad arguments");
    if (sm_count <= 0) {
        const int rc = q4::sm_count(&sm_count);
        if (rc != LF_OK) return rc;
    }
    // Pages are split until there are about eight items an SM, down to one page for each warp.
    const long own = max_pages - num_prefix_pages;
    int pps = 128;
    while (pps > 4 && (long)num_seqs * num_kv_heads * ((own + pps - 1) / pps) < 8L * sm_count) pps /= 2;
    *pages_per_split = pps;
    clear_error();
    return LF_OK;
}

extern "C" int lf_q4_decode_workspace_size(int num_seqs, int num_q_heads, int head_dim, int max_pages,
                                           int pages_per_split, int num_prefix_pages, size_t* bytes) {
    LF_CHECK_ARG(bytes != nullptr, "q4 decode: bytes is null");
    LF_CHECK_ARG(num_seqs >= 0 && num_q_heads > 0 && head_dim > 0 && max_pages > 0 && pages_per_split > 0 &&
                     num_prefix_pages >= 0 && num_prefix_pages <= max_pages,
                 "q4 decode: bad workspace arguments");
    *bytes = (size_t)num_seqs * num_q_heads * q4::slots_bound(max_pages, num_prefix_pages, pages_per_split) *
             ((size_t)head_dim * sizeof(float) + sizeof(float2));
    clear_error();
    return LF_OK;
}

extern "C" int lf_q4_decode_fwd(const lf_bf16* q, const void* pages, const int32_t* block_table,
                                const int32_t* seq_lens, int num_prefix_pages, lf_bf16* o, float* lse,
                                void* workspace, size_t workspace_bytes, int num_seqs, int num_q_heads,
                                int num_kv_heads, int head_dim, int num_pages, int max_pages,
                                int pages_per_split, float scale, void* stream) {
    LF_CHECK_ARG(num_seqs >= 0, "q4 decode: negative sizes");
    if (num_seqs == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(q && pages && block_table && seq_lens && o && workspace, "q4 decode: null pointer argument");
    LF_CHECK_ARG(aligned16(q) && aligned16(pages) && aligned16(o) && aligned16(workspace),
                 "q4 decode: q, pages, o and workspace must be 16-byte aligned");
    LF_CHECK_ARG(head_dim == 128 || head_dim == 64, "q4 decode: head_dim must be 64 or 128 (got %d)", head_dim);
    LF_CHECK_ARG(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
                 "q4 decode: need Hq a multiple of Hkv");
    const int G = num_q_heads / num_kv_heads;
    LF_CHECK_ARG(G == 1 || G == 2 || G == 4 || G == 8, "q4 decode: Hq/Hkv must be 1, 2, 4 or 8 (got %d)", G);
    LF_CHECK_ARG(num_pages > 0 && max_pages > 0 && max_pages <= (1 << 26) && pages_per_split > 0,
                 "q4 decode: num_pages, max_pages and pages_per_split must be > 0");
    LF_CHECK_ARG(num_prefix_pages >= 0 && num_prefix_pages <= max_pages,
                 "q4 decode: num_prefix_pages out of range");
    size_t need = 0;
    lf_q4_decode_workspace_size(num_seqs, num_q_heads, head_dim, max_pages, pages_per_split,
                                num_prefix_pages, &need);
    LF_CHECK_ARG(workspace_bytes >= need, "q4 decode: workspace too small (%zu < %zu bytes)", workspace_bytes, need);
    int sms = 0;
    const int rc = q4::sm_count(&sms);
    if (rc != LF_OK) return rc;
    q4::DecodeArgs a{};
    a.q = q;
    a.pages = static_cast<const uint8_t*>(pages);
    a.bt = block_table;
    a.lens = seq_lens;
    a.N = num_seqs;
    a.Hq = num_q_heads;
    a.Hkv = num_kv_heads;
    a.G = G;
    a.num_pages = num_pages;
    a.max_pages = max_pages;
    a.n_prefix = num_prefix_pages;
    a.chunk = q4::prefix_chunk(num_seqs, G, num_kv_heads, num_prefix_pages, sms);
    a.n_chunks = q4::ceil_div(num_prefix_pages, a.chunk);
    a.groups = q4::ceil_div(num_seqs, q4::kWarps * (8 / G));
    a.pps = pages_per_split;
    a.max_split = q4::own_splits(max_pages, num_prefix_pages, pages_per_split);
    a.n_slots = a.max_split + a.n_chunks;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)num_seqs * num_q_heads * a.n_slots * head_dim);
    a.qscale = scale * kLog2e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return head_dim == 128 ? q4::launch<128>(a, o, lse, st) : q4::launch<64>(a, o, lse, st);
}
