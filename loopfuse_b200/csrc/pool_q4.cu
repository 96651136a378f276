// Appending K/V to 4-bit pages, and expanding 4-bit pages to bf16 pages for the prefill kernel.
//
// Both are passes over memory: the append reads each new K/V value once and writes 4.5 bits of it, the
// expansion reads 4.5 bits and writes 16.  3796 tokens of 32 q and 8 k/v heads of 128: the append takes 28 us
// (82 MB; issue slots and latencies, 150 instructions a row pair), the expansion of their 32 sessions'
// contexts 58 us (280 MB, 4.8 TB/s).  The format is described in q4_common.cuh.
#include "pool_common.cuh"
#include "q4_common.cuh"
#include "sm100_primitives.cuh"

#include <math.h>

namespace lf {
namespace q4 {

constexpr uint32_t kSigns = 0x80008000u;
constexpr float kMagic = 12582912.f;                   // 1.5 * 2^23
constexpr uint32_t kMagicBits = 0x4B400000u;
constexpr float kSmallest = 1e-27f;                    // about 2^-90: smaller scales divide plainly

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Both halves of a bf16 pair as fp32.
__device__ __forceinline__ uint64_t pair_of(uint32_t w) { return sm100::f2_pack(bf16lo_to_f32(w), bf16hi_to_f32(w)); }

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t q_token, kv_layer, kv_token, kv_head;      // strides in elements
    const int32_t *table, *seq_ids, *start, *cu;
    int table_rows, table_stride, n, total;
    const float *cos, *sin;
    int rope_rows;
    uint16_t* q_out;
    uint8_t* pages;
    int num_pages, Hq, Hkv;
    int32_t* status;                                   // a pool's sticky status, or null
};

__device__ __forceinline__ void report(const AppendArgs& a) {
    if (a.status != nullptr) atomicCAS(a.status, LF_OK, LF_EINVAL);
    else atomicCAS(&g_device_error, 0, 252);
}

// One CTA walks tokens (grid-stride, blockIdx.y the layer); a row of D dims of one head is D / 8
// lanes of 8 dims: the queries' rows, then k's and v's, from the last warp on.  Rotation uses the partner
// lane's 8 dims and rounds every product and sum separately, then to bf16, as an eager fp32
// evaluation does; the codes are those of the rounded values.  A row that has no session, no page, or no
// rotation table row is not stored and is reported.
template <int D>
__global__ void __launch_bounds__(512, 2) append_kernel(const AppendArgs a) {
    using F = Fmt<D>;
    constexpr int LPR = D / 8, RPW = 32 / LPR;          // lanes a row, rows a warp
    grid_wait();
    if (a.status != nullptr && *reinterpret_cast<volatile int32_t*>(a.status) != LF_OK) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int l = lane % LPR, row0 = warp * RPW + lane / LPR;   // this lane's first query row
    const int kv0 = (warps - 1 - warp) * RPW + lane / LPR;      // and k or v row: the last warps begin
    const int H2 = 2 * a.Hkv, skip = warps * RPW;
    const long layer = blockIdx.y;
    for (int t = blockIdx.x; t < a.total; t += gridDim.x) {
        // This lane's first rows are on their way while the token is looked up.
        const uint16_t* qs = a.q + t * a.q_token + (long)row0 * D + 8 * l;
        auto source = [&](int h) -> const uint16_t* {           // k rows, then v rows
            const bool v = h >= a.Hkv;
            return (v ? a.v : a.k) + layer * a.kv_layer + t * a.kv_token + (h - (v ? a.Hkv : 0)) * a.kv_head + 8 * l;
        };
        uint4 q_next = make_uint4(0, 0, 0, 0), kv_next = q_next;
        if (row0 < a.Hq) q_next = *reinterpret_cast<const uint4*>(qs);
        if (kv0 < H2) kv_next = *reinterpret_cast<const uint4*>(source(kv0));
        int lo = 0;                                    // the last session i with cu[i] <= t, 32 probes at a time
        for (int len = a.n; len > 1;) {
            const int step = (len + 31) / 32, i = lo + lane * step;
            const bool below = lane * step < len && a.cu[i] <= t;
            const int k = max(0, 31 - __clz(__ballot_sync(0xffffffffu, below)));
            lo += k * step;
            len = min(step, len - k * step);
        }
        const int begin = a.cu[lo];
        const bool owned = t >= begin && t < a.cu[lo + 1];     // (no: before the first session or behind the last)
        const int pos = owned ? a.start[lo] + (t - begin) : -1;
        const int row = a.seq_ids != nullptr ? a.seq_ids[lo] : lo;
        const bool pos_ok = owned && (a.cos == nullptr || (pos >= 0 && pos < a.rope_rows));
        int page = -1;
        if (row >= 0 && row < a.table_rows && pos >= 0 && pos / kPage < a.table_stride)
            page = a.table[(long)row * a.table_stride + pos / kPage];
        const bool page_ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages);
        if (!(page_ok && pos_ok) && threadIdx.x == 0) report(a);
        float cs[8], sn[8];                            // this lane's dims, the same in every row: -s, s by half
        if (a.cos != nullptr) {
            const long off = (long)(pos_ok ? pos : 0) * (D / 2) + (8 * l) % (D / 2);
            const float sign = l < LPR / 2 ? -1.f : 1.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4 c = reinterpret_cast<const float4*>(a.cos + off)[j];
                const float4 n = reinterpret_cast<const float4*>(a.sin + off)[j];
                cs[4 * j] = c.x; cs[4 * j + 1] = c.y; cs[4 * j + 2] = c.z; cs[4 * j + 3] = c.w;
                sn[4 * j] = sign * n.x; sn[4 * j + 1] = sign * n.y;
                sn[4 * j + 2] = sign * n.z; sn[4 * j + 3] = sign * n.w;
            }
        }
        // x1 c - x2 s in the first half of a row, x2 c + x1 s in the second; a warp's lanes together.
        auto rotate = [&](uint32_t (&w)[4], bool turn) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t o = __shfl_xor_sync(0xffffffffu, w[j], LPR / 2);
                // (scalar: a packed multiplication and addition may be fused)
                const float lo = __fadd_rn(__fmul_rn(bf16lo_to_f32(w[j]), cs[2 * j]), __fmul_rn(bf16lo_to_f32(o), sn[2 * j]));
                const float hi = __fadd_rn(__fmul_rn(bf16hi_to_f32(w[j]), cs[2 * j + 1]), __fmul_rn(bf16hi_to_f32(o), sn[2 * j + 1]));
                if (turn) w[j] = pack_bf16x2(lo, hi);
            }
        };
        uint16_t* qd = a.q_out + ((long)t * a.Hq + row0) * D + 8 * l;
        for (int h = row0, r0 = warp * RPW; r0 < a.Hq; r0 += skip, h += skip) {
            uint32_t w[4] = {q_next.x, q_next.y, q_next.z, q_next.w};
            qs += skip * D;
            if (h + skip < a.Hq) q_next = *reinterpret_cast<const uint4*>(qs);
            if (a.cos != nullptr) rotate(w, true);
            if (h < a.Hq && pos_ok) *reinterpret_cast<uint4*>(qd) = make_uint4(w[0], w[1], w[2], w[3]);
            qd += skip * D;
        }
        for (int h = kv0, r0 = (warps - 1 - warp) * RPW; r0 < H2; r0 += skip, h += skip) {
            const bool live = h < H2, is_k = h < a.Hkv;
            const int kh = h - (is_k ? 0 : a.Hkv);
            uint32_t w[4] = {kv_next.x, kv_next.y, kv_next.z, kv_next.w};
            kv_next = make_uint4(0, 0, 0, 0);
            if (h + skip < H2) kv_next = *reinterpret_cast<const uint4*>(source(h + skip));
            if (a.cos != nullptr && __any_sync(0xffffffffu, is_k)) rotate(w, is_k);
            // {-min, max} of the group (8 lanes) as a bf16 pair, NaN if it holds one
            uint32_t ext;
            {
                const uint32_t hi = max2(max2(w[0], w[1]), max2(w[2], w[3]));
                const uint32_t lo = max2(max2(w[0] ^ kSigns, w[1] ^ kSigns), max2(w[2] ^ kSigns, w[3] ^ kSigns));
                ext = max2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
                for (int off = 1; off < 8; off <<= 1) ext = max2(ext, __shfl_xor_sync(0xffffffffu, ext, off));
            }
            if (!live || !page_ok || !pos_ok) continue;
            const float mn = -bf16lo_to_f32(ext), span = __fsub_rn(bf16hi_to_f32(ext), mn);
            uint32_t par = 0x7FC07FC0u;                // NaN, NaN
            uint32_t n[8];                             // the codes plus kMagicBits
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = kMagicBits;
            if (span < kMaxSpan) {                     // (not NaN)
                par = pack_bf16x2(__fdiv_rn(span, 15.f), mn);
                const float s = bf16lo_to_f32(par);
                uint64_t d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = sm100::fadd2(pair_of(w[j]), sm100::f2_pack(-mn, -mn));
                if (s >= kSmallest) {
                    // d / s rounded to nearest from the rounded reciprocal and the exact remainder of the
                    // first quotient (Markstein's theorem).  s is off by 2^-8 of itself at most, so d / s
                    // is at most 15 (1 + 2^-8) < 15.06 and rounds to 15 without a limit: adding 1.5 * 2^23
                    // leaves rint(d / s), ties to even, in the low bits.
                    const float r = __frcp_rn(s);
                    const uint64_t r2 = sm100::f2_pack(r, r), s2 = sm100::f2_pack(-s, -s), m2 = sm100::f2_pack(kMagic, kMagic);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint64_t q0 = fmul2(d[j], r2);
                        const float2 q1 = sm100::f2_unpack(sm100::fadd2(sm100::ffma2(sm100::ffma2(q0, s2, d[j]), r2, q0), m2));
                        n[2 * j] = __float_as_uint(q1.x);
                        n[2 * j + 1] = __float_as_uint(q1.y);
                    }
                } else if (s > 0.f) {                  // remainders would underflow
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 x = sm100::f2_unpack(d[j]);
                        n[2 * j] = __float_as_uint(__fadd_rn(fminf(rintf(__fdiv_rn(x.x, s)), 15.f), kMagic));
                        n[2 * j + 1] = __float_as_uint(__fadd_rn(fminf(rintf(__fdiv_rn(x.y, s)), 15.f), kMagic));
                    }
                }
            }
            const int tok = pos % kPage, grp = l / 8, in = l % 8;   // group, 8-dim piece of it
            uint8_t* blk = a.pages + ((layer * a.num_pages + page) * a.Hkv + kh) * (long)F::kBlockBytes;
            if (is_k) {                                // sums modulo 2^32; the magic bits' sum goes off
                uint32_t word = 0, magic = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t at = 1u << (4 * (e / 2) + 16 * (e % 2));
                    word += n[e] * at;
                    magic += kMagicBits * at;
                }
                *reinterpret_cast<uint32_t*>(blk + tok * (32 * F::NG) + (in / 2) * (8 * F::NG) +
                                             grp * 8 + (in % 2) * 4) = word - magic;
            } else {
                uint8_t* vp = blk + F::kVOff + (tok / 8) * (256 * F::NG) +
                              (in * 4 + (tok % 8) / 2) * (8 * F::NG) + grp * 8 + (tok % 2) * 2;
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    *reinterpret_cast<uint16_t*>(vp + 4 * q) = (uint16_t)(
                        n[4 * q] + n[4 * q + 1] * 16u + n[4 * q + 2] * 256u + n[4 * q + 3] * 4096u -
                        kMagicBits * 0x1111u);
            }
            if (in == 0)
                *reinterpret_cast<uint32_t*>(blk + F::kParOff + ((tok * 2 + (is_k ? 0 : 1)) * F::NG + grp) * 4) = par;
        }
    }
}

// -- expansion --------------------------------------------------------------------------------------
constexpr int kExpWarps = 8;
constexpr int kExpPages = 2;                           // table columns a CTA expands (8: 101 against 93 us)

// The pair of codes at bits 0..3 of both halves, as values: n s + b rounded once to bf16.  128 + n is put
// together from bits and 128 taken off again, both exact.
__device__ __forceinline__ uint32_t values(uint32_t w, uint32_t s2, uint32_t b2) {
    uint32_t n, r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(n) : "r"(w), "n"(0x000F000F), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(n) : "r"(n), "r"(0x43004300u));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(n), "r"(s2), "r"(b2));
    return r;
}

// CTA (session n, kExpPages columns of its table row): warps take (page, head) pairs.  Output pages
// are compact: the shared prefix first, then every session's own pages in session order; each CTA
// finds its session's first one by summing the lengths before it.  Rows at or past the length
// become zeros, so that the prefill kernel's masked products see no stale bits.
template <int D>
__global__ void __launch_bounds__(32 * kExpWarps)
expand_kernel(const uint8_t* pages, const int32_t* bt, const int32_t* lens, uint16_t* ko, uint16_t* vo,
              int32_t* out_table, int N, int Hkv, int num_pages, int max_pages,
              int n_prefix, int out_pages) {
    using F = Fmt<D>;
    grid_wait();
    const int chunks = (max_pages + kExpPages - 1) / kExpPages;
    const int n = blockIdx.x / chunks, j0 = (blockIdx.x % chunks) * kExpPages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto held = [&](int i) { return min(max(lens[i], 0), max_pages * kPage); };
    int own = 0, best = -1, best_n = 0;                // pages before this session's; longest session
    for (int i = threadIdx.x; i < N; i += 32 * kExpWarps) {
        const int L = held(i);
        if (i < n) own += max(0, (L + kPage - 1) / kPage - n_prefix);
        if (L > best) { best = L; best_n = i; }
    }
    __shared__ int s_own[kExpWarps], s_best[kExpWarps], s_arg[kExpWarps];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        own += __shfl_xor_sync(0xffffffffu, own, off);
        const int ob = __shfl_xor_sync(0xffffffffu, best, off), oa = __shfl_xor_sync(0xffffffffu, best_n, off);
        if (ob > best || (ob == best && oa < best_n)) { best = ob; best_n = oa; }
    }
    if (lane == 0) { s_own[warp] = own; s_best[warp] = best; s_arg[warp] = best_n; }
    __syncthreads();
    own = 0;
    best = -1;
    best_n = 0;
#pragma unroll
    for (int w = 0; w < kExpWarps; ++w) {
        own += s_own[w];
        if (s_best[w] > best || (s_best[w] == best && s_arg[w] < best_n)) { best = s_best[w]; best_n = s_arg[w]; }
    }
    const int L = held(n), np = (L + kPage - 1) / kPage;
    const int j_end = min(j0 + kExpPages, max_pages);
    auto out_page = [&](int j) { return j < n_prefix ? j : n_prefix + own + (j - n_prefix); };
    if (threadIdx.x < j_end - j0) {
        const int j = j0 + threadIdx.x;
        const int o = out_page(j);
        const bool fits = o < out_pages;
        out_table[(long)n * max_pages + j] = (j < np || j < n_prefix) && fits ? o : -1;
        if (j < np && !fits) atomicCAS(&g_device_error, 0, 253);
    }
    // shared pages are written once, from the longest session's row
    const int lead = best_n;
    const int g = lane >> 2, c = lane & 3;
    constexpr int NW = 2 * F::NG;                      // code words of a lane's vector
    // Pages this CTA writes: its own ones, and, in the lead session, the shared ones.
    const int j_last = min(j_end, max(np, n == lead ? n_prefix : 0));
    const int j_first = n == lead ? j0 : max(j0, n_prefix);
    const int units = max(0, j_last - j_first) * Hkv;
    for (int u = warp; u < units; u += kExpWarps) {
        const int j = j_first + u / Hkv, h = u % Hkv;
        const int o = out_page(j);
        if (o >= out_pages) break;
        const int rows = min(kPage, L - j * kPage);     // <= 0: a prefix page past every session
        int page = rows > 0 ? bt[(long)n * max_pages + j] : 0;
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(num_pages)) {
            if (lane == 0) atomicCAS(&g_device_error, 0, 254);
            page = 0;
        }
        const uint8_t* blk = pages + ((long)page * Hkv + h) * F::kBlockBytes;
        const long dst = ((long)o * Hkv + h) * (kPage * D);
        uint32_t kw[2][NW], vw[2][NW], pk[2][F::NG], pv[2][2][F::NG];
        const uint32_t* par = reinterpret_cast<const uint32_t*>(blk + F::kParOff);
#pragma unroll
        for (int half = 0; half < 2; ++half) {         // all loads before the first use
            const uint8_t* kp = blk + (half * 8 + g) * (32 * F::NG) + c * (8 * F::NG);
            const uint8_t* vp = blk + F::kVOff + half * (256 * F::NG) + lane * (8 * F::NG);
            if constexpr (F::NG == 2) {
                const uint4 a = ld_stream(kp), b = ld_stream(vp);
                kw[half][0] = a.x; kw[half][1] = a.y; kw[half][2] = a.z; kw[half][3] = a.w;
                vw[half][0] = b.x; vw[half][1] = b.y; vw[half][2] = b.z; vw[half][3] = b.w;
            } else {
                const uint2 a = *reinterpret_cast<const uint2*>(kp);
                const uint2 b = *reinterpret_cast<const uint2*>(vp);
                kw[half][0] = a.x; kw[half][1] = a.y;
                vw[half][0] = b.x; vw[half][1] = b.y;
            }
#pragma unroll
            for (int grp = 0; grp < F::NG; ++grp) {
                pk[half][grp] = par[(half * 8 + g) * 2 * F::NG + grp];
                pv[half][0][grp] = par[((half * 8 + 2 * c) * 2 + 1) * F::NG + grp];
                pv[half][1][grp] = par[((half * 8 + 2 * c) * 2 + 3) * F::NG + grp];
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int t = half * 8 + g;                // K: the lane's 16 dims of a group, 32 bytes
#pragma unroll
            for (int grp = 0; grp < F::NG; ++grp) {
                uint32_t out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (t < rows) {
                    const uint32_t p = pk[half][grp];
                    const uint32_t s2 = __byte_perm(p, p, 0x1010), b2 = __byte_perm(p, p, 0x3232);
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[4 * w + i] = values(kw[half][2 * grp + w] >> (4 * i), s2, b2);
                }
                sm100::st_global_v8(ko + dst + t * D + grp * kGroup + c * 16, out);
            }
            // V: tokens t0, t0 + 1 (a word's halves), 8 dims of a group, 16 bytes each
            const int t0 = half * 8 + 2 * c;
#pragma unroll
            for (int grp = 0; grp < F::NG; ++grp) {
                const uint32_t p0 = pv[half][0][grp], p1 = pv[half][1][grp];
                const uint32_t s2 = __byte_perm(p0, p1, 0x5410), b2 = __byte_perm(p0, p1, 0x7632);
                uint32_t even[4], odd[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {          // dims 2 i, 2 i + 1 of both tokens
                    const uint32_t w = vw[half][2 * grp + i / 2] >> (8 * (i % 2));
                    const uint32_t x = values(w, s2, b2), y = values(w >> 4, s2, b2);
                    even[i] = t0 < rows ? __byte_perm(x, y, 0x5410) : 0u;
                    odd[i] = t0 + 1 < rows ? __byte_perm(x, y, 0x7632) : 0u;
                }
                uint16_t* to = vo + dst + t0 * D + grp * kGroup + g * 8;
                *reinterpret_cast<uint4*>(to) = make_uint4(even[0], even[1], even[2], even[3]);
                *reinterpret_cast<uint4*>(to + D) = make_uint4(odd[0], odd[1], odd[2], odd[3]);
            }
        }
    }
}

// The rows a fork needs of a session's partial last page: whole blocks are copied (rows past the
// prefix are overwritten by the destination's own tokens before anything reads them).
__global__ void fork_copy_kernel(const int32_t* __restrict__ status, const int32_t* __restrict__ bt,
                                 int table_stride, int table_rows, int src, const int32_t* __restrict__ dsts,
                                 int full, uint8_t* __restrict__ pages, int num_pages, long page_bytes) {
    if (*reinterpret_cast<const volatile int32_t*>(status) != LF_OK) return;
    const int d = dsts[blockIdx.x];
    if (d < 0 || d >= table_rows) return;
    const int sp = bt[(long)src * table_stride + full], dp = bt[(long)d * table_stride + full];
    if (static_cast<unsigned>(sp) >= static_cast<unsigned>(num_pages) ||
        static_cast<unsigned>(dp) >= static_cast<unsigned>(num_pages))
        return;
    const uint4* from = reinterpret_cast<const uint4*>(pages + ((long)blockIdx.y * num_pages + sp) * page_bytes);
    uint4* to = reinterpret_cast<uint4*>(pages + ((long)blockIdx.y * num_pages + dp) * page_bytes);
    for (long i = threadIdx.x; i < page_bytes / 16; i += blockDim.x) to[i] = from[i];
}

}  // namespace q4
}  // namespace lf

using namespace lf;

extern "C" int lf_q4_append(const lf_bf16* q, const lf_bf16* k, const lf_bf16* v,
                            int64_t q_stride_token, int64_t stride_layer, int64_t stride_token,
                            int64_t stride_head, const int32_t* block_table, int table_rows,
                            int max_pages, const int32_t* seq_ids, const int32_t* start_pos,
                            const int32_t* cu_tokens, int n, int total_tokens, const float* rope_cos,
                            const float* rope_sin, int rope_rows, lf_bf16* q_out, void* pages,
                            int num_pages, int num_layers, int num_q_heads, int num_kv_heads,
                            int head_dim, int32_t* status, void* stream) {
    LF_CHECK_ARG(n >= 0 && total_tokens >= 0, "q4 append: negative sizes");
    if (n == 0 || total_tokens == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(k && v && block_table && start_pos && cu_tokens && pages, "q4 append: null pointer argument");
    LF_CHECK_ARG(head_dim == 64 || head_dim == 128, "q4 append: head_dim must be 64 or 128 (got %d)", head_dim);
    LF_CHECK_ARG(num_q_heads >= 0 && num_kv_heads > 0 && num_pages > 0 && max_pages > 0 && max_pages <= (1 << 26) && table_rows > 0 &&
                     num_layers > 0 && num_layers <= 65535,
                 "q4 append: bad shape");
    LF_CHECK_ARG(num_q_heads == 0 || (q && q_out && num_layers == 1), "q4 append: q needs q_out and one layer");
    LF_CHECK_ARG(seq_ids != nullptr || n <= table_rows, "q4 append: more sessions than block-table rows");
    LF_CHECK_ARG(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(pages) &&
                     q_stride_token % 8 == 0 && stride_layer % 8 == 0 && stride_token % 8 == 0 &&
                     stride_head % 8 == 0,
                 "q4 append: rows and pages must be 16-byte aligned");
    LF_CHECK_ARG((rope_cos == nullptr) == (rope_sin == nullptr), "q4 append: give cos and sin");
    LF_CHECK_ARG(rope_cos == nullptr || (rope_rows > 0 && aligned16(rope_cos) && aligned16(rope_sin)),
                 "q4 append: rope tables must be 16-byte aligned with rows > 0");
    const q4::AppendArgs a{q, k, v, q_stride_token, stride_layer, stride_token, stride_head, block_table,
                           seq_ids, start_pos, cu_tokens, table_rows, max_pages, n, total_tokens, rope_cos,
                           rope_sin, rope_rows, q_out, static_cast<uint8_t*>(pages), num_pages, num_q_heads,
                           num_kv_heads, status};
    const int rows = num_q_heads + 2 * num_kv_heads, rpw = 256 / head_dim;
    // A token's rows are spread over 16 warps while there are few tokens, over 2 once the tokens fill
    // the chip by themselves (what a warp looks up once per token then serves more rows).
    const int warps = (rows + rpw - 1) / rpw, most = total_tokens >= 148 * 4 ? 2 : 16;
    const int threads = 32 * (warps < most ? warps : most);
    const int blocks = total_tokens < 148 * 32 ? total_tokens : 148 * 32;
    const dim3 grid(blocks, num_layers);
    return launch_early("q4 append", head_dim == 128 ? q4::append_kernel<128> : q4::append_kernel<64>, grid,
                        dim3(threads), 0, (cudaStream_t)stream, a);
}

extern "C" int lf_q4_expand(const void* pages, const int32_t* block_table, const int32_t* seq_lens,
                            int num_prefix_pages, lf_bf16* k_out, lf_bf16* v_out, int32_t* out_table,
                            int num_seqs, int num_kv_heads, int head_dim, int num_pages, int max_pages,
                            int out_pages, void* stream) {
    LF_CHECK_ARG(num_seqs >= 0, "q4 expand: negative sizes");
    if (num_seqs == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(pages && block_table && seq_lens && out_table && out_pages >= 0 &&
                     (out_pages == 0 || (k_out && v_out)),
                 "q4 expand: null pointer argument");
    LF_CHECK_ARG(head_dim == 64 || head_dim == 128, "q4 expand: head_dim must be 64 or 128 (got %d)", head_dim);
    LF_CHECK_ARG(num_kv_heads > 0 && num_pages > 0 && max_pages > 0 && max_pages <= (1 << 26) &&
                     num_prefix_pages >= 0 && num_prefix_pages <= max_pages,
                 "q4 expand: bad shape");
    LF_CHECK_ARG(aligned16(pages) && (reinterpret_cast<uintptr_t>(k_out) & 31u) == 0 && aligned16(v_out),
                 "q4 expand: pages and v_out must be 16-byte aligned, k_out 32-byte aligned");
    const long blocks = (long)num_seqs * ((max_pages + q4::kExpPages - 1) / q4::kExpPages);
    LF_CHECK_ARG(blocks <= 2147483647L, "q4 expand: grid limits exceeded");
    return launch_early("q4 expand", head_dim == 128 ? q4::expand_kernel<128> : q4::expand_kernel<64>,
                        dim3((unsigned)blocks), dim3(32 * q4::kExpWarps), 0, (cudaStream_t)stream,
                        static_cast<const uint8_t*>(pages), block_table, seq_lens, k_out, v_out, out_table, num_seqs,
                        num_kv_heads, num_pages, max_pages, num_prefix_pages, out_pages);
}

extern "C" int lf_q4_fork(const lf_pool_meta* m, int src_seq, const int32_t* dst_seqs, int n,
                          int prefix_len, void* pages, int num_layers, int num_kv_heads, int head_dim,
                          void* stream) {
    LF_CHECK_ARG(pages != nullptr && aligned16(pages) && num_layers > 0 && num_layers <= 65535 &&
                     num_kv_heads > 0 && (head_dim == 64 || head_dim == 128),
                 "q4 fork: bad data arguments");
    const int rc = lf_pool_fork(m, src_seq, dst_seqs, n, prefix_len, nullptr, nullptr, 0, 0, 8, stream);
    if (rc != LF_OK || n == 0 || prefix_len % LF_PAGE_SIZE == 0) return rc;
    LF_CHECK_ARG(src_seq >= 0 && src_seq < m->max_seqs && prefix_len > 0 &&
                     prefix_len <= m->max_pages_per_seq * LF_PAGE_SIZE,
                 "q4 fork: bad source or prefix");
    q4::fork_copy_kernel<<<dim3(n, num_layers), 256, 0, (cudaStream_t)stream>>>(
        m->ctrl + LF_CTRL_STATUS, m->block_table, m->max_pages_per_seq, m->max_seqs, src_seq, dst_seqs,
        prefix_len / LF_PAGE_SIZE, static_cast<uint8_t*>(pages), m->num_pages,
        (long)num_kv_heads * 18 * head_dim);
    return launch_status("q4 fork copy");
}
