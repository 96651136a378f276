// Log probabilities of given tokens, the entropy of each distribution and its top alternatives, from
// a batch of logits rows, in one pass over them.
//
// Per row, with m = max x:  s = sum e^(x - m),  w = sum e^(x - m) (x - m),
//   log p(token) = (x_token - m) - ln s,   entropy = ln s - w / s,
// and the k largest logits, ties to the lowest index.  w is taken around the running maximum, so that
// a peaked distribution's small entropy is not a difference of large numbers; -inf logits (banned
// tokens) enter both sums as zeros.
//
// Work is bound by reading the logits: at 2 bytes a value an SM receives about 12 values a clock, and
// can issue 128 lane-instructions.  So the sums are kept in the log2 domain,
//   t = (x - m) log2 e,  s = sum 2^t,  w = sum 2^t t,
// on packed pairs of fp32 (two values an instruction), -inf being raised to a finite value first:
// about 5 instructions a value, one of them the exponential.  Maxima are taken on packed 16-bit pairs.
// x - m, not a multiply-add with a rounded m log2 e: a certain token's t is exactly 0.
// A row is taken by a cluster of 1 to 8 CTAs, so that small batches fill the chip; a warp takes slices
// of 8 vectors of 16 bytes per lane, and 32 warps an SM keep loads in flight under each other's
// arithmetic.  (Loading a slice ahead in registers leaves room for fewer warps: 78 against 73 us for
// 1501 rows of 128256 bf16.)  Every lane keeps its own (m, s, w) and rescales once a slice.
//
// The alternatives are found among whole vectors: the k vectors with the largest maxima (ties to the
// lowest index) hold the k largest values, since a value of any other vector is beaten by each of
// their k maxima.  A warp keeps its best vectors as a sorted list, lane i the i-th as a 64-bit key
// (maximum, then lowest index); it starts from the lanes' best vectors of the first slice, and a
// later slice is searched only when some lane's maximum reaches the list's k-th.  Lists are merged by
// bitonic exchanges, in the CTA through shared memory and in the cluster through distributed shared
// memory, and the values of the last k vectors are read again, each counting those above it: one launch,
// no workspace, no atomics, the same result in every run.  64 rows of 128256 bf16 (16 MB, in L2): 12.9 us
// with 20 alternatives, 6.5 without any; one row 7.9 and 3.6.
#include "lf_common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

namespace lf {
namespace logprobs {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kVecs = 8;                               // 16-byte vectors of a lane's slice
constexpr int kPerSm = 4;                              // resident CTAs of an SM
constexpr int kMaxParts = 8;                           // CTAs of a row (portable cluster size)
constexpr unsigned kAll = 0xffffffffu;

typedef unsigned long long u64;
constexpr float kHuge = 1.3e36f;                       // 2^120: maxima past it are far from the type's end

template <int DT> struct Elem;                         // 0 bf16, 1 fp16, 2 fp32
template <> struct Elem<0> {
    typedef uint16_t T;
    static constexpr int N = 8;
    static constexpr uint32_t kNegInf = 0xFF80FF80u;
    static constexpr uint32_t kFloor = 0xFE80FE80u;    // -2^126
    static constexpr float kLowest = -1.3e36f;         // maxima from here on are far above the floor
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = bf16lo_to_f32(w); f[1] = bf16hi_to_f32(w); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
template <> struct Elem<1> {
    typedef uint16_t T;
    static constexpr int N = 8;
    static constexpr uint32_t kNegInf = 0xFC00FC00u;
    static constexpr uint32_t kFloor = 0xFBFFFBFFu;    // -65504
    static constexpr float kLowest = -60000.f;
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
        f[0] = v.x;
        f[1] = v.y;
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
template <> struct Elem<2> {
    typedef uint32_t T;
    static constexpr int N = 4;
    static constexpr uint32_t kNegInf = 0xFF800000u;
    static constexpr uint32_t kFloor = 0xFE800000u;    // -2^126
    static constexpr float kLowest = -1.3e36f;
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Packed pairs of fp32.
__device__ __forceinline__ u64 pair(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(u64 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Largest of a vector's values (NaN if one is).
template <int DT>
__device__ __forceinline__ float vec_max(const uint4& v) {
    if constexpr (DT == 2) {
        return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                       max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
        float f[2];
        Elem<DT>::unpack(Elem<DT>::max2(Elem<DT>::max2(v.x, v.y), Elem<DT>::max2(v.z, v.w)), f);
        return max_nan(f[0], f[1]);
    }
}

// The values of a vector, in order.
template <int DT>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[Elem<DT>::N]) {
    constexpr int P = Elem<DT>::N / 4;
    Elem<DT>::unpack(v.x, f);
    Elem<DT>::unpack(v.y, f + P);
    Elem<DT>::unpack(v.z, f + 2 * P);
    Elem<DT>::unpack(v.w, f + 3 * P);
}

// Keys order by value (NaN above all, both zeros alike), then by lowest index; 0 is below every key.
__device__ __forceinline__ u64 make_key(float x, uint32_t index) {
    uint32_t b = __float_as_uint(x + 0.f);             // -0 + 0 = +0
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    if (x != x) b = 0xFFFFFFFFu;
    return ((u64)b << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(u64 k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }

// Sorts a bitonic sequence over the lanes, largest first.
__device__ __forceinline__ u64 bitonic_merge(u64 k, int lane) {
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) {
        const u64 o = __shfl_xor_sync(kAll, k, j);
        const bool upper = (lane & j) == 0;            // keeps the larger
        k = ((o > k) == upper) ? o : k;
    }
    return k;
}
__device__ __forceinline__ u64 sort_desc(u64 k, int lane) {
#pragma unroll
    for (int size = 2; size < 32; size <<= 1)
#pragma unroll
        for (int j = size >> 1; j > 0; j >>= 1) {
            const u64 o = __shfl_xor_sync(kAll, k, j);
            const bool upper = ((lane & j) == 0) == ((lane & size) == 0);
            k = ((o > k) == upper) ? o : k;
        }
    return bitonic_merge(k, lane);
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ u64 merge_lists(u64 a, u64 b, int lane) {
    const u64 r = __shfl_sync(kAll, b, 31 - lane);
    return bitonic_merge(a > r ? a : r, lane);
}

struct Stat {                                          // of a set of values: maximum, sums around it
    float m, s, w;
    // The sums around a larger maximum.
    __device__ __forceinline__ void raise(float m2) {
        const float d = fmaxf((m - m2) * kLog2e, -1e30f);   // finite: from -inf, s and w are 0
        const float f = fast_exp2(d);
        w = f * (w + d * s);
        s *= f;
        m = m2;
    }
};
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float m = max_nan(a.m, b.m);
    if (m != a.m) a.raise(m);
    if (m != b.m) b.raise(m);
    return Stat{m, a.s + b.s, a.w + b.w};
}

struct Args {
    const void* x;
    int64_t stride;                                    // elements
    const void* tokens;
    int tokens64, vocab, k, parts;
    float *logprob, *entropy;
    int64_t* ids;
    float* top;
};

__device__ __forceinline__ int64_t token(const Args& a, long row) {
    return a.tokens64 ? static_cast<const int64_t*>(a.tokens)[row] : (int64_t)static_cast<const int32_t*>(a.tokens)[row];
}

template <int DT, bool kTop>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_kernel(const Args a) {
    using E = Elem<DT>;
    typedef typename E::T T;
    constexpr int N = E::N;
    constexpr uint32_t kSlice = 32u * N * kVecs;       // values of a warp's slice
    __shared__ __align__(16) u64 s_list[kWarps][32];
    __shared__ Stat s_stat[kWarps];
    __shared__ u64 c_list[kMaxParts][32];              // the cluster's, in its first CTA
    __shared__ Stat c_stat[kMaxParts];
    const int part = blockIdx.x % a.parts;
    const long row = blockIdx.x / a.parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    // Positions u = v + lead count from the 16-byte boundary at or before the row, so that vectors
    // are aligned; the row is [lead, end).
    const uint32_t lead = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const uint32_t end = lead + (uint32_t)a.vocab;
    const T* base = x - lead;
    const uint32_t slices = (end + kSlice - 1) / kSlice;
    const uint32_t per = (slices + a.parts - 1) / a.parts;
    const uint32_t s_end = min(slices, (part + 1) * per);

    auto load = [&](uint32_t slice, uint4 (&v)[kVecs]) {
        const uint32_t u0 = slice * kSlice + lane * N;
        if (slice * kSlice >= lead && (slice + 1) * kSlice <= end) {   // warp-uniform: whole slice
#pragma unroll
            for (int i = 0; i < kVecs; ++i) v[i] = ld_stream(base + u0 + i * 32 * N);
            return;
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const uint32_t u = u0 + i * 32 * N;
            uint32_t w[4] = {E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
            if (u >= lead && u + N <= end) {
                v[i] = ld_stream(base + u);
                continue;
            }
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (u + e >= lead && u + e < end) {
                    if constexpr (DT == 2) w[e] = base[u + e];
                    else w[e / 2] = (w[e / 2] & (e % 2 ? 0x0000FFFFu : 0xFFFF0000u)) | ((uint32_t)base[u + e] << (16 * (e % 2)));
                }
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };

    __shared__ float s_tok;
    if (a.parts > 1) cluster_arrive();                 // waited for before the first remote store
    grid_wait();
    if (part == 0 && threadIdx.x == kThreads - 1) {    // the token's own logit, on its way meanwhile
        const int64_t tok = token(a, row);
        float f[2] = {0.f, 0.f};
        if (tok >= 0 && tok < a.vocab) E::unpack((uint32_t)x[tok], f);
        s_tok = f[0];
    }
    Stat st{-INFINITY, 0.f, 0.f};
    u64 list = 0, kth = 0, own = 0;                    // this lane's entry; the k-th entry
    float thr = -INFINITY;                             // no vector below it enters the list
    bool first = true;
    auto slice = [&](uint32_t sl, const uint4 (&cur)[kVecs]) {
        float vm[kVecs];
        float lm = -INFINITY;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            vm[i] = vec_max<DT>(cur[i]);
            lm = max_nan(lm, vm[i]);
        }
        if (!(lm <= st.m)) st.raise(max_nan(st.m, lm));
        const bool none = st.m == -INFINITY;           // every value so far is -inf: all terms are 0
        if (__all_sync(kAll, none || (st.m >= E::kLowest && st.m < kHuge))) {
            const float M = none ? 0.f : -st.m;
            const u64 M2 = pair(M, M), L2 = pair(kLog2e, kLog2e);
            u64 s2 = 0, w2 = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const uint32_t v[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
                float f[N];
#pragma unroll
                for (int e = 0; e < 4; ++e) E::unpack(E::max2(v[e], E::kFloor), f + e * (N / 4));
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const u64 t2 = mul2(add2(pair(f[e], f[e + 1]), M2), L2);
                    float t0, t1;
                    split(t2, t0, t1);
                    const u64 p2 = pair(fast_exp2(t0), fast_exp2(t1));
                    s2 = add2(s2, p2);
                    w2 = fma2(p2, t2, w2);
                }
            }
            float s0, s1, w0, w1;
            split(s2, s0, s1);
            split(w2, w0, w1);
            if (!none) {
                st.s += s0 + s1;
                st.w += w0 + w1;
            }
        } else if (!none) {                            // maxima out of range: differences, one by one
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                float f[N];
                unpack<DT>(cur[i], f);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float t = fmaxf((f[e] - st.m) * kLog2e, -1e30f);
                    const float p = fast_exp2(t);
                    st.s += p;
                    st.w = fmaf(p, t, st.w);
                }
            }
        }
        if constexpr (kTop) {
            const uint32_t v0 = sl * (kSlice / N) + lane;     // this lane's vectors: v0 + 32 i
            auto key_of = [&](int i) {                 // a vector without a value of the row has none
                const uint32_t v = v0 + 32 * i;
                return v * N + N > lead && v * N < end ? make_key(vm[i], v) : 0;
            };
            if (first) {                               // the list starts from the lanes' best vectors
                first = false;
                u64 best = 0;
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    const u64 k = key_of(i);
                    best = k > best ? k : best;
                }
                list = sort_desc(best, lane);
                kth = __shfl_sync(kAll, list, a.k - 1);
                own = best;
            }
            if (__any_sync(kAll, !(lm < thr))) {
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    u64 key = !(vm[i] < thr) ? key_of(i) : 0;
                    if (key == own) key = 0;           // in the list already
                    unsigned in = __ballot_sync(kAll, key > kth);
                    if (in == 0) continue;
                    if (__popc(in) > 6) {              // many at once: sort them and merge
                        list = merge_lists(list, sort_desc(key > kth ? key : 0, lane), lane);
                    } else {
                        while (in != 0) {
                            const u64 c = __shfl_sync(kAll, key, __ffs(in) - 1);
                            in &= in - 1;
                            const int pos = __popc(__ballot_sync(kAll, list > c));
                            const u64 up = __shfl_up_sync(kAll, list, 1);
                            list = lane < pos ? list : (lane == pos ? c : up);
                        }
                    }
                    kth = __shfl_sync(kAll, list, a.k - 1);
                }
                own = 0;
                if (kth != 0) {                        // a NaN there lets everything be looked at
                    const float v = key_value(kth);
                    thr = v != v ? -INFINITY : v;
                }
            }
        }
    };
    for (uint32_t sl = part * per + warp; sl < s_end; sl += kWarps) {
        uint4 v[kVecs];
        load(sl, v);
        slice(sl, v);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const Stat o{__shfl_xor_sync(kAll, st.m, off), __shfl_xor_sync(kAll, st.s, off),
                     __shfl_xor_sync(kAll, st.w, off)};
        st = merge(st, o);
    }
    // A tree over lists in shared memory, halving the number of lists: warp i takes i and i + half.
    auto tree = [&](u64 (*lists)[32], Stat* stats, int count) {
        for (int n = count; n > 1; n = (n + 1) / 2) {
            const int half = (n + 1) / 2;
            __syncthreads();
            if (warp < n - half) {
                if (kTop) lists[warp][lane] = merge_lists(lists[warp][lane], lists[warp + half][lane], lane);
                const Stat r = merge(stats[warp], stats[warp + half]);
                __syncwarp();
                if (lane == 0) stats[warp] = r;
            }
        }
        __syncthreads();
    };
    if (kTop) s_list[warp][lane] = list;
    if (lane == 0) s_stat[warp] = st;
    tree(s_list, s_stat, kWarps);
    u64(*lists)[32] = s_list;
    Stat* stats = s_stat;
    if (a.parts > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster_wait();                                // the first CTA runs
        if (warp == 0) {
            if (kTop) *cluster.map_shared_rank(&c_list[part][lane], 0) = s_list[0][lane];
            if (lane == 0) *cluster.map_shared_rank(&c_stat[part], 0) = s_stat[0];
        }
        cluster.sync();
        if (part != 0) return;
        lists = c_list;
        stats = c_stat;
        tree(lists, stats, a.parts);
    }
    if (warp != 0) return;
    st = stats[0];
    const bool none = st.m == -INFINITY, bad = !(st.m < INFINITY);
    const float ln_s = none || bad ? 0.f : logf(st.s);
    auto logp = [&](float v) { return bad ? NAN : (none ? -INFINITY : (v - st.m) - ln_s); };
    if (kTop) {
        // The values of the k best vectors that reach the k-th vector's maximum hold the k best values
        // (at least k do); they are packed, and each counts those above it.
        const u64 mine = lists[0][lane];
        const bool have = mine != 0 && lane < a.k;
        const uint32_t u = key_index(mine) * N;
        const u64 last = __shfl_sync(kAll, mine, a.k - 1);   // 0: fewer than k vectors
        const float bar = last == 0 ? -INFINITY : key_value(last);
        float val[N];
        unsigned in = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t p = u + e;
            float f[2] = {-INFINITY, 0.f};
            const bool inside = have && p >= lead && p < end;
            if (inside) E::unpack((uint32_t)base[p], f);
            val[e] = f[0];
            in |= (inside && !(f[0] < bar) ? 1u : 0u) << e;
        }
        int at = __popc(in);                           // where this lane's begin
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(kAll, at, off);
            if (lane >= off) at += o;
        }
        const int n = __shfl_sync(kAll, at, 31);       // at most 32 N
        at -= __popc(in);
        static_assert(kWarps * 32 >= 32 * N, "room for the candidates");
        u64* cand = &s_list[0][0];                     // (the lists have been read)
        __syncwarp();
#pragma unroll
        for (int e = 0; e < N; ++e)
            if ((in >> e) & 1u) cand[at++] = make_key(val[e], u + e - lead);
        if (lane == 0 && (n & 1)) cand[n] = 0;
        __syncwarp();
        for (int c = lane; c < n; c += 32) {
            const u64 key = cand[c];
            int pos = 0;
#pragma unroll 8
            for (int j = 0; j < n; j += 2) {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(cand + j);
                pos += (o.x > key) + (o.y > key);
            }
            if (pos < a.k) {
                a.ids[row * a.k + pos] = (int64_t)key_index(key);
                a.top[row * a.k + pos] = logp(key_value(key));
            }
        }
    }
    if (lane == 0) {
        const int64_t tok = token(a, row);
        if (tok >= a.vocab) atomicCAS(&g_device_error, 0, 231);
        // a negative token: none was given
        a.logprob[row] = tok < 0 ? 0.f : (tok >= a.vocab ? NAN : logp(s_tok));
        a.entropy[row] = bad ? NAN : (none ? 0.f : ln_s - st.w / st.s * kLn2);
    }
}

template <int DT>
static int launch(const Args& a, int rows, cudaStream_t st) {
    return launch_early_clusters("token logprobs", a.k > 0 ? logprobs_kernel<DT, true> : logprobs_kernel<DT, false>, a.parts,
                                 dim3((unsigned)((long)rows * a.parts)), dim3(kThreads), 0, st, a);
}

}  // namespace logprobs
}  // namespace lf

using namespace lf;

extern "C" int lf_token_logprobs(const void* logits, int dtype, int64_t row_stride, const void* tokens,
                                 int tokens_64bit, int rows, int vocab, int top_k, float* logprob,
                                 float* entropy, int64_t* top_ids, float* top_logprobs, void* stream) {
    LF_CHECK_ARG(rows >= 0 && vocab > 0, "token logprobs: rows >= 0 and vocab > 0 are needed");
    LF_CHECK_ARG(dtype >= 0 && dtype <= 2, "token logprobs: dtype must be LF_BF16, LF_FP16 or LF_FP32");
    LF_CHECK_ARG(top_k >= 0 && top_k <= 32 && top_k <= vocab, "token logprobs: top_k must be 0..32 and at most vocab");
    LF_CHECK_ARG(vocab <= (1 << 30), "token logprobs: vocab too large");
    LF_CHECK_ARG(rows <= 1 || row_stride >= vocab, "token logprobs: rows overlap");
    if (rows == 0) { clear_error(); return LF_OK; }
    LF_CHECK_ARG(logits && tokens && logprob && entropy && (top_k == 0 || (top_ids && top_logprobs)),
                 "token logprobs: null pointer argument");
    LF_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % (dtype == 2 ? 4 : 2) == 0, "token logprobs: unaligned logits");
    int dev = 0, sms = 0;
    LF_CHECK_CUDA(cudaGetDevice(&dev));
    LF_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // CTAs of a row: doubled while all of them stay resident at once and a warp keeps a slice
    const int slice = 32 * logprobs::kVecs * (dtype == 2 ? 4 : 8);
    int parts = 1;
    while (parts < logprobs::kMaxParts && 2L * rows * parts <= (long)logprobs::kPerSm * sms &&
           (long)vocab > (long)parts * logprobs::kWarps * slice)
        parts *= 2;
    LF_CHECK_ARG((long)rows * parts <= 2147483647L, "token logprobs: grid limits exceeded");
    const logprobs::Args a{logits, row_stride, tokens, tokens_64bit != 0, vocab, top_k, parts,
                           logprob, entropy, top_ids, top_logprobs};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 0) return logprobs::launch<0>(a, rows, st);
    if (dtype == 1) return logprobs::launch<1>(a, rows, st);
    return logprobs::launch<2>(a, rows, st);
}
