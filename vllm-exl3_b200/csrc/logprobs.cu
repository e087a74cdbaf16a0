// logprobs.cu -- per row of logits x: log p(token), entropy, the token's rank
// and the `top` best alternatives, in one pass.
//
// With m a running maximum and d_i = x_i - m:
//   s = sum exp d_i,  w = sum d_i exp d_i,
//   log p(t) = d_t - log s,  H = log s - w / s;
// (m, s, w) of two parts join by rescaling.  rank = 1 + #{x_i > x_t} + #{i < t: x_i = x_t}.
//
// Bound: every logit is read once: HBM (bf16: about 12 logits per clock and SM
// at the measured copy rate, near the 16 per clock of the exponential unit).
// A CTA streams a slice of one row, each thread 4 16-byte vectors at a time
// with the next 4 on their way (cp.async: 64 KB per SM without a register).  A
// thread's reference m follows its maximum only when that has grown by more
// than 4, so that the loop has next to no dependent rescaling.  A sum whose
// reference lies D below its largest entry carries that entry's roundings D
// times into H, and its weight's error into log p; so the lag is kept small, and
// after the loop each thread brings its sums to its largest entry, by the
// reciprocal of the very weight that the entry was given.  The entry then weighs
// 1, joins keep the largest entry, s >= 1, log p <= 0 and H >= 0, and a confident
// token's log p has the digits of a plain fp32 softmax (an entry 10 above the best of
// 131071 others: log p to 1e-7, with a lag of 16 and without this to 1.1e-6).
// Cost: 64 rows with 5 alternatives 15.0 -> 15.6 us, 2048 rows 124.6 -> 125.7;
// a lag of 8 would take 125.0.
// Few rows: a row is split over CTAs and joined by the one that ends last,
// always in the same order.
//
// Alternatives: entries are ordered by a 64-bit key (value, then lowest index
// first).  The `top`-th largest of 32 thread groups' maxima bounds the answer
// from below, so only the few threads whose maximum passes it have candidates;
// all warps then read those threads' entries again (from L2) and collect what
// passes, some `top` entries.  The buffer holds whatever one such round can
// yield; before it could overflow (many ties) it is reduced, which raises the bound.
//
// Measured: 2048 rows of 131072 bf16 104 us in a graph, 119 to 126 as a lone call
// from HBM, by the card (4.3 to 4.5 TB/s, 66 to 69 % of the measured copy rate;
// exponential unit and ALU are at 68 and 58 % of their rates); 64 rows with 5
// alternatives 15.4 us, 14.2 in a graph, one row of 100277 f32 with 20
// alternatives 12.5 us (pass, join, selection one after another).
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "exl3_common.cuh"

namespace exl3 {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpUnroll = 4;     // vectors of a thread in work
constexpr int kLpStages = 2;     // such sets in shared memory, on their way (3: 102.5 us where 2 take 100.8)
constexpr int kLpMaxTop = 32;    // one group maximum each
constexpr int kLpRound = kLpThreads * 8;               // most entries that one round of candidates looks at
constexpr int kLpCap = kLpRound + 2 * kLpMaxTop;       // candidate keys a CTA holds
constexpr float kLpSlack = 4.f;                        // growth of the maximum that the reference lets pass
constexpr int kLpMaxSplit = 64;
static_assert(kLpMaxSplit * kLpMaxTop <= kLpCap, "the parts' lists are joined in one buffer");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LpArgs {
    const char* x;
    int64_t stride;  // bytes
    int64_t rows;
    int vocab;
    const void* tokens;
    int ids_dtype;
    int top, splits;
    float *logprob, *entropy;
    int32_t* rank;
    float* top_logprobs;
    int32_t* top_ids;
    int32_t* counters;
    float4* stats;   // [rows][splits] {m, s, w, count}
    uint64_t* keys;  // [rows][splits][top]
};

struct LpStats {
    float m, s, w;  // m = -inf: nothing but -inf so far
    int above;
};

__device__ __forceinline__ void lp_join(LpStats& a, const LpStats& b) {
    const float m = fmaxf(a.m, b.m);
    auto bring = [m](const LpStats& p, float& s, float& w) {
        const float d = p.m == m ? 0.f : p.m - m;
        const float f = ex2(d * kLog2e);
        s = p.s * f;
        w = f == 0.f ? 0.f : (p.w + p.s * d) * f;
    };
    float sa, wa, sb, wb;
    bring(a, sa, wa);
    bring(b, sb, wb);
    a.m = m, a.s = sa + sb, a.w = wa + wb, a.above += b.above;
}

__device__ __forceinline__ void lp_join_warp(LpStats& st) {
    #pragma unroll
    for (int d = 16; d; d >>= 1)
        lp_join(st, LpStats{__shfl_xor_sync(0xffffffffu, st.m, d), __shfl_xor_sync(0xffffffffu, st.s, d),
                            __shfl_xor_sync(0xffffffffu, st.w, d), __shfl_xor_sync(0xffffffffu, st.above, d)});
}

__device__ __forceinline__ uint32_t sortable(float x) {  // ascending; NaN as -inf, -0 as 0
    const uint32_t b = __float_as_uint(x == x ? x + 0.f : -INFINITY);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_sortable(uint32_t k) {
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// Keeps the `top` largest of keys[0, n) in keys[0, top), descending.  All
// threads; keys are distinct.
__device__ __forceinline__ void lp_reduce(uint64_t* keys, uint64_t* best, int n, int top) {
    for (int i = threadIdx.x; i < n; i += kLpThreads) {
        const uint64_t k = keys[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += keys[j] > k;
        if (r < top) best[r] = k;
    }
    __syncthreads();
    if (threadIdx.x < min(n, top)) keys[threadIdx.x] = best[threadIdx.x];
    __syncthreads();
}

template <int DT>
struct LpType {
    static constexpr int kVec = DT == DT_F32 ? 4 : 8;
    static constexpr int kSize = DT == DT_F32 ? 4 : 2;
    // element i of a 16-byte vector
    static __device__ __forceinline__ float get(const uint4& v, int i) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (DT == DT_F32) return __uint_as_float(w[i]);
        else if constexpr (DT == DT_BF16) return __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
            return (i & 1) ? __high2float(h) : __low2float(h);
        }
    }
    static __device__ __forceinline__ uint32_t word(const uint4& v, int i) {
        return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    }
    static __device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
    static __device__ __forceinline__ __nv_bfloat162 b2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    static __device__ __forceinline__ float largest(const uint4& v) {  // NaN left out unless all are
        if constexpr (DT == DT_F32) {
            return fmaxf(fmaxf(get(v, 0), get(v, 1)), fmaxf(get(v, 2), get(v, 3)));
        } else if constexpr (DT == DT_BF16) {
            const __nv_bfloat162 m = __hmax2(__hmax2(b2(v.x), b2(v.y)), __hmax2(b2(v.z), b2(v.w)));
            return fmaxf(__low2float(m), __high2float(m));
        } else {
            const __half2 m = __hmax2(__hmax2(h2(v.x), h2(v.y)), __hmax2(h2(v.z), h2(v.w)));
            return fmaxf(__low2float(m), __high2float(m));
        }
    }
    // A reference this near 0 is far above the lowest number: their difference has weight 0 and is finite.
    static constexpr float kNear = DT == DT_F16 ? 3e4f : 1e35f;
    // entries 2 i and 2 i + 1, -inf as the lowest number
    static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
        if constexpr (DT == DT_F32) {
            return make_float2(max_nan(get(v, 2 * i), -3.3e38f), max_nan(get(v, 2 * i + 1), -3.3e38f));
        } else if constexpr (DT == DT_BF16) {
            const __nv_bfloat162 x = __hmax2_nan(b2(word(v, i)), b2(0xff7fff7fu));
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&x);
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        } else {
            return __half22float2(__hmax2_nan(h2(word(v, i)), h2(0xfbfffbffu)));
        }
    }
    // Entries above a threshold: of 16-bit types counted two at a time, as sums of ones
    using Count = std::conditional_t<DT == DT_F32, int, std::conditional_t<DT == DT_F16, __half2, __nv_bfloat162>>;
    using Level = std::conditional_t<DT == DT_F32, float, uint32_t>;
    static __device__ __forceinline__ Count zero() {
        if constexpr (DT == DT_F32) return 0;
        else if constexpr (DT == DT_F16) return h2(0u);
        else return b2(0u);
    }
    static __device__ __forceinline__ Level level(float x) {  // exact: x is an entry, or infinite
        if constexpr (DT == DT_F32) {
            return x;
        } else if constexpr (DT == DT_F16) {
            const __half2 t = __float2half2_rn(x);
            return *reinterpret_cast<const uint32_t*>(&t);
        } else {
            const __nv_bfloat162 t = __float2bfloat162_rn(x);
            return *reinterpret_cast<const uint32_t*>(&t);
        }
    }
    // the next lower number of the type, so that x >= t is x > below(t); t > -inf
    static __device__ __forceinline__ Level below(Level t) {
        if constexpr (DT == DT_F32) {
            const uint32_t b = __float_as_uint(t);
            return __uint_as_float((b & 0x7fffffffu) == 0u ? 0x80000001u : b >> 31 ? b + 1 : b - 1);
        } else {
            uint32_t b = t & 0xffffu;
            b = (b & 0x7fffu) == 0u ? 0x8001u : b >> 15 ? b + 1 : b - 1;
            return b | (b << 16);
        }
    }
    static __device__ __forceinline__ void count(Count& n, const uint4& v, Level t) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == DT_F32) n += get(v, i) > t;
            else if constexpr (DT == DT_F16) n = __hadd2(n, __hgt2(h2(word(v, i)), h2(t)));
            else n = __hadd2(n, __hgt2(b2(word(v, i)), b2(t)));
        }
    }
    static __device__ __forceinline__ int total(Count n) {
        if constexpr (DT == DT_F32) return n;
        else return int(__low2float(n)) + int(__high2float(n));
    }
    static __device__ __forceinline__ float at(const char* x, int64_t i) { return load_as_float(x, i, DT); }
    static constexpr uint32_t kNone = DT == DT_F32 ? 0xff800000u : DT == DT_F16 ? 0xfc00fc00u : 0xff80ff80u;  // -inf
};

template <int DT, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const LpArgs a) {
    using T = LpType<DT>;
    constexpr int VEC = T::kVec, U = kLpUnroll;
    extern __shared__ __align__(16) uint4 lp_ring[];                  // [kLpStages][U][threads]
    uint64_t* cand = reinterpret_cast<uint64_t*>(lp_ring);            // [kLpCap], once the ring is done with
    uint64_t* best = cand + kLpCap;                                   // [kLpMaxSplit], at least kLpMaxTop
    __shared__ uint32_t group_max[32];
    __shared__ uint16_t flagged[kLpThreads];
    __shared__ float wr[kLpWarps], ws[kLpWarps], ww[kLpWarps];
    __shared__ int wc[kLpWarps];
    __shared__ int count, n_flagged, last_flag;
    __shared__ uint64_t bound;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.splits;
    const int split = int(blockIdx.x % a.splits);
    const char* x = a.x + row * a.stride;
    const int64_t tok = load_id(a.tokens, row, a.ids_dtype);
    const bool asked = tok >= 0 && tok < a.vocab;
    const float xt = asked ? T::at(x, tok) : INFINITY;  // nothing ranks above +inf

    // The row: `head` entries up to the first 16-byte boundary, n_vec whole vectors, the rest.  This
    // CTA's vectors are [v0, v1); the first part has the head too, the last one the rest.
    const int head = min(int((-reinterpret_cast<uintptr_t>(x) & 15) / T::kSize), a.vocab);
    const int n_vec = (a.vocab - head) / VEC, rest = (a.vocab - head) % VEC;
    const uint4* vecs = reinterpret_cast<const uint4*>(x + head * T::kSize);
    const int v0 = int(int64_t(n_vec) * split / a.splits), v1 = int(int64_t(n_vec) * (split + 1) / a.splits);
    // index of this thread's single entry, one of the at most 2 (VEC - 1) at the ends, or -1
    int single = -1;
    if (split == 0 && tid < head) single = tid;
    if (split == a.splits - 1 && tid >= 32 && tid < 32 + rest) single = a.vocab - rest + tid - 32;

    // rank: entries before the token count when as high, the others when higher; entries of the
    // token's own vector, and single ones, are looked at one by one
    const bool lowest = xt == -INFINITY;  // every entry before it counts, seen or not
    const auto above_t = T::level(xt), from_t = lowest ? T::level(INFINITY) : T::below(above_t);
    const int tok_vec = !asked ? -1 : tok < head ? -1 : int((tok - head) / VEC);

    LpStats st{-INFINITY, 0.f, 0.f, 0};
    float mx_all = -INFINITY;
    if (single >= 0) {
        const float v = T::at(x, single);
        const bool fine = v < INFINITY;  // NaN and +inf make the row NaN
        st.m = fine ? v : 0.f, st.s = fine ? (v == -INFINITY ? 0.f : 1.f) : NAN, st.w = fine ? 0.f : NAN;
        if (asked && !(lowest && single < tok)) st.above += v > xt || (v == xt && single < tok);
        mx_all = v == v ? v : -INFINITY;
    }
    if (asked && split == 0 && tid == 0 && lowest) st.above += int(tok);
    if (asked && tok_vec >= v0 && tok_vec < v1 && tid >= 64 && tid < 64 + VEC) {
        const int i = head + tok_vec * VEC + tid - 64;  // before it, in its vector, whose entries above it the loop counts
        const float v = T::at(x, i);
        if (i < tok) st.above += lowest ? -int(v > xt) : int(v == xt);
    }

    // a thread's vectors go through places of its own in shared memory: no barrier
    const uint32_t ring = smem_u32(lp_ring) + tid * 16;
    auto fetch = [&](int j, int stage) {
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * kLpThreads < v1)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(ring + (stage * U + u) * (kLpThreads * 16)),
                             "l"(vecs + j + u * kLpThreads) : "memory");
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    #pragma unroll
    for (int i = 0; i < kLpStages - 1; ++i) fetch(v0 + i * U * kLpThreads + tid, i);
    int stage = 0;
    #pragma unroll 1
    for (int j0 = v0; j0 < v1; j0 += U * kLpThreads) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(kLpStages - 2) : "memory");
        uint4 v[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) v[u] = lp_ring[(stage * U + u) * kLpThreads + tid];
        fetch(j0 + (kLpStages - 1) * U * kLpThreads + tid, stage == 0 ? kLpStages - 1 : stage - 1);
        stage = stage == kLpStages - 1 ? 0 : stage + 1;
        if (j0 + U * kLpThreads > v1) {
            #pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + tid + u * kLpThreads >= v1) v[u] = make_uint4(T::kNone, T::kNone, T::kNone, T::kNone);
        }
        float mx = T::largest(v[0]);
        #pragma unroll
        for (int u = 1; u < U; ++u) mx = fmaxf(mx, T::largest(v[u]));
        mx_all = fmaxf(mx_all, mx);
        if (mx > st.m + kLpSlack || (st.m == -INFINITY && mx > st.m)) lp_join(st, LpStats{mx, 0.f, 0.f, 0});
        const float ref = st.m == -INFINITY ? 0.f : st.m;
        if (fabsf(ref) < T::kNear) {
            // two at a time.  -inf stands as the type's lowest number: its weight is 0 against such
            // a reference, and 0 times the difference stays 0
            const float2 neg = make_float2(-ref, -ref), l2 = make_float2(kLog2e, kLog2e);
            float2 s2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
            #pragma unroll
            for (int u = 0; u < U; ++u)
                #pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    const float2 d = add2(T::pair(v[u], i), neg);
                    const float2 t = mul2(d, l2);
                    const float2 e = make_float2(ex2(t.x), ex2(t.y));
                    s2 = add2(s2, e);
                    w2 = fma2(e, d, w2);
                }
            st.s += s2.x + s2.y, st.w += w2.x + w2.y;
        } else {
            #pragma unroll
            for (int u = 0; u < U; ++u)
                #pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = max_nan(T::get(v[u], i) - ref, -300.f);
                    const float e = ex2(d * kLog2e);
                    st.s += e;
                    st.w = fmaf(e, d, st.w);
                }
        }
        typename T::Count n = T::zero();
        #pragma unroll
        for (int u = 0; u < U; ++u) T::count(n, v[u], j0 + tid + u * kLpThreads < tok_vec ? from_t : above_t);
        st.above += T::total(n);
    }

    // --- alternatives ---
    if constexpr (TOP) {
        const uint32_t own = sortable(mx_all);
        uint32_t gm = own;
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 1));
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
        if ((lane & 7) == 0) group_max[tid >> 3] = gm;
        if (tid == 0) count = 0, n_flagged = 0, bound = 0;
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        __syncthreads();
        if (warp == 0) {
            const uint32_t g = group_max[lane];
            int rank = 0;
            #pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t o = __shfl_sync(0xffffffffu, g, i);
                rank += o > g || (o == g && i < lane);
            }
            if (rank == a.top - 1) bound = uint64_t(g) << 32;  // every key of the value g is above this
        }
        __syncthreads();
        if (own >= uint32_t(bound >> 32)) flagged[atomicAdd(&n_flagged, 1)] = uint16_t(tid);
        if (single >= 0) {
            const uint64_t key = (uint64_t(sortable(T::at(x, single))) << 32) | (0xffffffffu - uint32_t(single));
            if (key > bound) cand[atomicAdd(&count, 1)] = key;
        }
        __syncthreads();
        // 32 vectors of 8 flagged threads a round: a warp to each
        const int per = (v1 - v0 + kLpThreads - 1) / kLpThreads, rounds = (per + 31) / 32;
        for (int f0 = 0; f0 < n_flagged; f0 += kLpWarps) {
            for (int k = 0; k < rounds; ++k) {
                const int n = count;
                __syncthreads();
                if (n > kLpCap - kLpRound) {
                    lp_reduce(cand, best, n, a.top);
                    if (tid == 0) {
                        count = min(n, a.top);
                        if (n >= a.top) bound = max(bound, cand[a.top - 1]);
                    }
                    __syncthreads();
                }
                const uint64_t least = bound;
                const int j = f0 + warp < n_flagged ? v0 + flagged[f0 + warp] + (32 * k + lane) * kLpThreads : v1;
                if (j < v1) {
                    const uint4 v = __ldg(vecs + j);
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const uint64_t key = (uint64_t(sortable(T::get(v, i))) << 32) | (0xffffffffu - uint32_t(head + j * VEC + i));
                        if (key > least) cand[atomicAdd(&count, 1)] = key;
                    }
                }
                __syncthreads();
            }
        }
        lp_reduce(cand, best, count, a.top);
    }

    // --- join the threads, each at its largest entry ---
    {
        const float to = fmaxf(mx_all, st.m), d = to == st.m ? 0.f : to - st.m, f = __fdividef(1.f, ex2(d * kLog2e));
        st.w = fmaf(-st.s, d, st.w) * f, st.s *= f, st.m = to;
    }
    lp_join_warp(st);
    if (lane == 0) wr[warp] = st.m, ws[warp] = st.s, ww[warp] = st.w, wc[warp] = st.above;
    __syncthreads();
    st = LpStats{wr[0], ws[0], ww[0], wc[0]};
    for (int w = 1; w < kLpWarps; ++w) lp_join(st, LpStats{wr[w], ws[w], ww[w], wc[w]});
    const int have = TOP ? min(count, a.top) : 0;

    if (a.splits > 1) {
        const int64_t slot = row * a.splits + split;
        if (tid == 0) __stcg(a.stats + slot, make_float4(st.m, st.s, st.w, __int_as_float(st.above)));
        for (int i = tid; i < a.top; i += kLpThreads) __stcg(a.keys + slot * a.top + i, i < have ? cand[i] : 0);
        __syncthreads();
        if (tid == 0) {
            int prev;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(a.counters + row) : "memory");
            last_flag = prev == a.splits - 1;
            if (prev == a.splits - 1) a.counters[row] = 0;  // ready for the next call
        }
        __syncthreads();
        if (!last_flag) return;
        // lane i takes parts i and i + 32, then the lanes join: the same order every time
        st = LpStats{-INFINITY, 0.f, 0.f, 0};
        for (int i = lane; i < a.splits; i += 32) {
            const float4 o = __ldcg(a.stats + row * a.splits + i);
            lp_join(st, LpStats{o.x, o.y, o.z, __float_as_int(o.w)});
        }
        lp_join_warp(st);
        if constexpr (TOP) {
            // The lists are in order.  With c + 1 the keys of a list that are surely enough from m
            // lists, c = ceil(top / splits) - 1, m = ceil(top / (c + 1)): the m-th largest of the
            // lists' c-th keys bounds the answer from below, and little more than `top` keys pass it.
            const int c = (a.top - 1) / a.splits, m = (a.top + c) / (c + 1);
            const uint64_t* keys = a.keys + row * a.splits * a.top;
            if (tid < a.splits) best[tid] = __ldcg(keys + tid * a.top + c);
            if (tid == 0) count = 0, bound = 0;
            __syncthreads();
            if (tid < a.splits) {
                int n = 0;
                for (int i = 0; i < a.splits; ++i) n += best[i] > best[tid] || (best[i] == best[tid] && i < tid);
                if (n == m - 1) bound = best[tid];
            }
            __syncthreads();
            const uint64_t least = max(bound, uint64_t(1));  // 0: no key
            for (int i = tid; i < a.splits * a.top; i += kLpThreads) {
                const uint64_t k = __ldcg(keys + i);
                if (k >= least) cand[atomicAdd(&count, 1)] = k;
            }
            __syncthreads();
            lp_reduce(cand, best, count, a.top);
        }
    }
    if (st.s > 0.f && st.s < 1.f) st.s = 1.f;  // the largest entry weighs 1: less is rounding
    const float ls = log2f(st.s) * kLn2;
    auto logp = [&](float v) { return st.s == 0.f ? -INFINITY : (v - st.m) - ls; };  // s = 0: a row of -inf
    if (tid == 0) {
        a.logprob[row] = asked ? logp(xt) : -INFINITY;
        const float h = st.s == 0.f ? 0.f : ls - st.w / st.s;
        a.entropy[row] = h < 0.f ? 0.f : h;
        a.rank[row] = asked ? 1 + st.above : 0;
    }
    for (int i = tid; i < a.top; i += kLpThreads) {
        const uint64_t k = cand[i];
        a.top_logprobs[row * a.top + i] = logp(from_sortable(uint32_t(k >> 32)));
        a.top_ids[row * a.top + i] = int32_t(0xffffffffu - uint32_t(k));
    }
}

// Over how many CTAs a row is split: as many as run at once (4 per SM), no
// less than two vectors a thread.  More rows than half of that are not split:
// the join costs more than the last wave's empty places (2048 rows of 131072
// bf16, 3.46 waves: 101 us whole, 117 us in halves).
static int lp_splits(const LogprobsCall& c, int sms) {
    const int64_t vectors = c.vocab / (c.x_dtype == DT_F32 ? 4 : 8);
    const int64_t want = 4 * int64_t(sms) / c.rows, most = vectors / (2 * kLpThreads);
    const int64_t n = want < most ? want : most;
    return int(n < 1 ? 1 : n > kLpMaxSplit ? kLpMaxSplit : n);
}

// one per row that can be split
int logprobs_counters(int sms) { return 2 * sms; }

size_t logprobs_workspace(const LogprobsCall& c, int sms) {
    const int splits = lp_splits(c, sms);
    return splits > 1 ? size_t(c.rows) * splits * (16 + 8 * size_t(c.top)) : 0;
}

template <int DT, bool TOP>
static cudaError_t launch_logprobs(const LpArgs& a, unsigned grid, cudaStream_t s) {
    constexpr size_t smem = size_t(kLpStages) * kLpUnroll * kLpThreads * 16;
    static_assert(smem >= size_t(kLpCap + kLpMaxSplit) * 8, "the candidates take the ring's place");
    auto* kernel = logprobs_kernel<DT, TOP>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = raise_smem(kernel, smem, done);
    if (e != cudaSuccess) return e;
    kernel<<<grid, kLpThreads, smem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t run_logprobs(const LogprobsCall& c, int sms, cudaStream_t s) {
    if (c.rows <= 0) return cudaSuccess;
    LpArgs a;
    a.x = static_cast<const char*>(c.logits), a.stride = c.stride * (c.x_dtype == DT_F32 ? 4 : 2);
    a.rows = c.rows, a.vocab = c.vocab, a.tokens = c.tokens, a.ids_dtype = c.ids_dtype;
    a.top = c.top, a.splits = lp_splits(c, sms);
    a.logprob = c.logprob, a.entropy = c.entropy, a.rank = c.rank;
    a.top_logprobs = c.top_logprobs, a.top_ids = c.top_ids, a.counters = c.counters;
    a.stats = reinterpret_cast<float4*>(c.ws);
    a.keys = reinterpret_cast<uint64_t*>(c.ws + size_t(c.rows) * a.splits * 16);
    const unsigned grid = unsigned(c.rows * a.splits);
    const auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return c.top ? launch_logprobs<DT, true>(a, grid, s) : launch_logprobs<DT, false>(a, grid, s);
    };
    if (c.x_dtype == DT_F32) return go(std::integral_constant<int, DT_F32>());
    if (c.x_dtype == DT_F16) return go(std::integral_constant<int, DT_F16>());
    return go(std::integral_constant<int, DT_BF16>());
}

}  // namespace exl3
