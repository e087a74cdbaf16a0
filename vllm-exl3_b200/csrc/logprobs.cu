// logprobs.cu -- per row of logits x: log p(token), entropy, the token's rank
// and the `top` best alternatives, in one pass.
//
// With m a running maximum and d_i = x_i - m:
//   s = sum exp d_i,  w = sum d_i exp d_i,
//   log p(t) = d_t - log s,  H = log s - w / s
// (H has no difference of large numbers); (m, s, w) of two parts join by
// rescaling.  rank = 1 + #{x_i > x_t} + #{i < t: x_i = x_t}.
//
// Bound: every logit is read once: HBM (bf16: about 12 logits per clock and SM
// at the measured copy rate, near the 16 per clock of the exponential unit).
// A CTA takes a slice of one row, in chunks that its threads hold in
// registers (16-byte loads, U of them in flight per thread), so a chunk's
// maximum is known before its exponentials are taken.  Few rows: a row
// is split over CTAs and joined by the one that ends last, in slice order.
//
// Alternatives: entries are ordered by a 64-bit key (value, then lowest index
// first).  The `top`-th largest of 32 group maxima of a chunk bounds the
// answer from below, so a chunk yields some `top` candidates, not thousands;
// they are collected in shared memory and reduced by counting, for each, the
// larger ones.  Where more tie or pass the bound than the buffer holds, the
// buffer is reduced, the bound rises, and the chunk is looked through again.
// The few threads whose maximum passes the bound read their entries again
// (from L1 or L2) rather than keep them in registers.
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "exl3_common.cuh"

namespace exl3 {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpCap = 2048;     // candidate keys a CTA holds
constexpr int kLpMaxTop = 32;    // one group maximum each
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
    int top, splits, chunks;  // chunks per row
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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

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
    // Counts: of 16-bit types two at a time, as sums of ones (at most 32 a half before total())
    using Count = std::conditional_t<DT == DT_F32, int, std::conditional_t<DT == DT_F16, __half2, __nv_bfloat162>>;
    static __device__ __forceinline__ Count zero() {
        if constexpr (DT == DT_F32) return 0;
        else if constexpr (DT == DT_F16) return h2(0u);
        else return b2(0u);
    }
    template <bool GE>
    static __device__ __forceinline__ void count(Count& n, const uint4& v, float xt) {
        if constexpr (DT == DT_F32) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) n += GE ? get(v, i) >= xt : get(v, i) > xt;
        } else {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == DT_F16) {
                    const __half2 t = __float2half2_rn(xt);  // exact: an entry of the row, or +inf
                    n = __hadd2(n, GE ? __hge2(h2(word(v, i)), t) : __hgt2(h2(word(v, i)), t));
                } else {
                    const __nv_bfloat162 t = __float2bfloat162_rn(xt);
                    n = __hadd2(n, GE ? __hge2(b2(word(v, i)), t) : __hgt2(b2(word(v, i)), t));
                }
            }
        }
    }
    static __device__ __forceinline__ void count_ge(Count& n, const uint4& v, float xt) { count<true>(n, v, xt); }
    static __device__ __forceinline__ void count_gt(Count& n, const uint4& v, float xt) { count<false>(n, v, xt); }
    static __device__ __forceinline__ int total(Count n) {
        if constexpr (DT == DT_F32) return n;
        else return int(__low2float(n)) + int(__high2float(n));
    }
};

template <int DT, int U, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const LpArgs a) {
    using T = LpType<DT>;
    constexpr int VEC = T::kVec;
    extern __shared__ uint64_t lp_smem[];
    uint64_t* cand = lp_smem;            // [kLpCap]
    uint64_t* best = lp_smem + kLpCap;   // [kLpMaxSplit], at least kLpMaxTop
    __shared__ uint32_t group_max[32];
    __shared__ float wr[kLpWarps], ws[kLpWarps], ww[kLpWarps];
    __shared__ int wc[kLpWarps];
    __shared__ int count, last_flag;
    __shared__ uint64_t bound;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.splits;
    const int split = int(blockIdx.x % a.splits);
    const char* x = a.x + row * a.stride;
    const int shift = int((reinterpret_cast<uintptr_t>(x) & 15) / T::kSize);  // entries of vector 0 before the row
    const char* base = x - shift * T::kSize;
    const int64_t tok = load_id(a.tokens, row, a.ids_dtype);
    const bool asked = tok >= 0 && tok < a.vocab;
    float xt = INFINITY;  // nothing ranks above it
    if (asked) xt = load_as_float(x, tok, DT);
    const int c0 = int(int64_t(a.chunks) * split / a.splits), c1 = int(int64_t(a.chunks) * (split + 1) / a.splits);

    LpStats st{-INFINITY, 0.f, 0.f, 0};
    if (tid == 0) count = 0, bound = 0;
    __syncthreads();

    // 16-byte vector j of the row, whose first entry has index e0
    auto load = [&](int64_t j, int64_t e0) {
        if (e0 >= 0 && e0 + VEC <= a.vocab) return __ldg(reinterpret_cast<const uint4*>(base) + j);
        uint32_t w[4];  // a row's ends: entry by entry, -inf outside
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == DT_F32) {
                const int64_t e = e0 + i;
                w[i] = e >= 0 && e < a.vocab ? reinterpret_cast<const uint32_t*>(x)[e] : 0xff800000u;
            } else {
                const uint32_t ninf = DT == DT_F16 ? 0xfc00u : 0xff80u;
                const int64_t e = e0 + 2 * i;
                const uint16_t* p = reinterpret_cast<const uint16_t*>(x);
                const uint32_t lo = e >= 0 && e < a.vocab ? p[e] : ninf;
                const uint32_t hi = e + 1 >= 0 && e + 1 < a.vocab ? p[e + 1] : ninf;
                w[i] = lo | (hi << 16);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };

    for (int c = c0; c < c1; ++c) {
        uint4 v[U];
        const int64_t j0 = int64_t(c) * U * kLpThreads + tid;
        float mx = -INFINITY;
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = j0 + u * kLpThreads;
            v[u] = load(j, j * VEC - shift);
        }
        #pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, T::largest(v[u]));

        // --- sums ---
        LpStats part{mx, 0.f, 0.f, 0};
        const float ref = mx == -INFINITY ? 0.f : mx;
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
            part.s = s2.x + s2.y, part.w = w2.x + w2.y;
        } else {
            #pragma unroll 1
            for (int u = 0; u < U; ++u) {
                const int64_t j = j0 + u * kLpThreads;
                const uint4 again = load(j, j * VEC - shift);
                #pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = max_nan(T::get(again, i) - ref, -300.f);
                    const float e = ex2(d * kLog2e);
                    part.s += e;
                    part.w = fmaf(e, d, part.w);
                }
            }
        }
        // --- rank: entries above the token, and before it as high ---
        typename T::Count before_n = T::zero(), after_n = T::zero();
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t e0 = (j0 + u * kLpThreads) * VEC - shift;
            if (e0 + VEC <= tok) {
                T::count_ge(before_n, v[u], xt);
                // entries before the row's first one are no part of it
                if (e0 < 0 && xt == -INFINITY) part.above += int(e0);
            } else if (e0 > tok) {
                T::count_gt(after_n, v[u], xt);
            } else {
                #pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xi = T::get(v[u], i);
                    part.above += xi > xt || (xi == xt && e0 + i >= 0 && e0 + i < tok);
                }
            }
        }
        part.above += T::total(before_n) + T::total(after_n);
        lp_join(st, part);

        // --- alternatives ---
        if constexpr (!TOP) continue;
        uint32_t gm = sortable(mx);
        if (!__syncthreads_or(gm >= uint32_t(bound >> 32))) continue;
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 1));
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
        gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
        if ((lane & 7) == 0) group_max[tid >> 3] = gm;
        __syncthreads();
        if (warp == 0) {
            const uint32_t g = group_max[lane];
            int r = 0;
            #pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t o = __shfl_sync(0xffffffffu, g, i);
                r += o > g || (o == g && i < lane);
            }
            if (r == a.top - 1) bound = max(bound, uint64_t(g) << 32);
        }
        __syncthreads();
        uint64_t pushed = 0;
        for (;;) {
            const uint64_t least = bound;
            const uint32_t least_hi = uint32_t(least >> 32);
            bool full = false;
            if (sortable(mx) >= least_hi) {
                #pragma unroll 1
                for (int u = 0; u < U; ++u) {
                    const int64_t j = j0 + u * kLpThreads, e0 = j * VEC - shift;
                    const uint4 again = load(j, e0);
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const uint32_t sv = sortable(T::get(again, i));
                        if (sv < least_hi || e0 + i < 0 || e0 + i >= a.vocab) continue;
                        const uint64_t key = (uint64_t(sv) << 32) | (0xffffffffu - uint32_t(e0 + i));
                        if (key <= least || (pushed >> (u * VEC + i) & 1)) continue;
                        const int at = atomicAdd(&count, 1);
                        if (at < kLpCap) cand[at] = key, pushed |= uint64_t(1) << (u * VEC + i);
                        else full = true;
                    }
                }
            }
            const bool again = __syncthreads_or(full);
            const int n = min(count, kLpCap);
            lp_reduce(cand, best, n, a.top);
            if (tid == 0) {
                count = min(n, a.top);
                // keys at or below the last of a full list cannot enter it
                if (n >= a.top) bound = max(bound, cand[a.top - 1]);
            }
            __syncthreads();
            if (!again) break;
        }
    }

    // --- join the threads ---
    lp_join_warp(st);
    if (lane == 0) wr[warp] = st.m, ws[warp] = st.s, ww[warp] = st.w, wc[warp] = st.above;
    __syncthreads();
    st = LpStats{wr[0], ws[0], ww[0], wc[0]};
    for (int w = 1; w < kLpWarps; ++w) lp_join(st, LpStats{wr[w], ws[w], ww[w], wc[w]});
    int have = a.top ? count : 0;

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
    const float ls = log2f(st.s) * kLn2;
    auto logp = [&](float v) { return st.s == 0.f ? -INFINITY : (v - st.m) - ls; };  // s = 0: a row of -inf
    if (tid == 0) {
        a.logprob[row] = asked ? logp(xt) : -INFINITY;
        a.entropy[row] = st.s == 0.f ? 0.f : ls - st.w / st.s;
        a.rank[row] = asked ? 1 + st.above : 0;
    }
    for (int i = tid; i < a.top; i += kLpThreads) {
        const uint64_t k = cand[i];
        a.top_logprobs[row * a.top + i] = logp(from_sortable(uint32_t(k >> 32)));
        a.top_ids[row * a.top + i] = int32_t(0xffffffffu - uint32_t(k));
    }
}

// A row's chunks of 256 threads x U vectors (one vector more than the row's
// own where its start is not aligned), and over how many CTAs it is split:
// what runs at once (4 CTAs per SM).
struct LpPlan {
    int U, chunks, splits;
};
static LpPlan lp_plan(const LogprobsCall& c, int sms) {
    const int vec = c.x_dtype == DT_F32 ? 4 : 8;
    auto chunks = [&](int U) { return int((c.vocab + vec - 1 + int64_t(vec) * kLpThreads * U - 1) / (int64_t(vec) * kLpThreads * U)); };
    // few rows: chunks of 2 vectors, so that a row spreads over four times the CTAs
    const int U = c.rows * chunks(8) < sms ? 2 : 8;
    LpPlan p{U, chunks(U), 1};
    const int64_t want = 4 * int64_t(sms) / c.rows;
    p.splits = int(want < 1 ? 1 : want < p.chunks ? want : p.chunks);
    if (p.splits > kLpMaxSplit) p.splits = kLpMaxSplit;
    return p;
}

// a row is split only where there are at most two rows per SM
int logprobs_counters(int sms) { return 2 * sms; }

size_t logprobs_workspace(const LogprobsCall& c, int sms) {
    const LpPlan p = lp_plan(c, sms);
    return p.splits > 1 ? size_t(c.rows) * p.splits * (16 + 8 * size_t(c.top)) : 0;
}

cudaError_t run_logprobs(const LogprobsCall& c, int sms, cudaStream_t s) {
    if (c.rows <= 0) return cudaSuccess;
    const LpPlan p = lp_plan(c, sms);
    LpArgs a;
    a.x = static_cast<const char*>(c.logits), a.stride = c.stride * (c.x_dtype == DT_F32 ? 4 : 2);
    a.rows = c.rows, a.vocab = c.vocab, a.tokens = c.tokens, a.ids_dtype = c.ids_dtype;
    a.top = c.top, a.splits = p.splits, a.chunks = p.chunks;
    a.logprob = c.logprob, a.entropy = c.entropy, a.rank = c.rank;
    a.top_logprobs = c.top_logprobs, a.top_ids = c.top_ids, a.counters = c.counters;
    a.stats = reinterpret_cast<float4*>(c.ws);
    a.keys = reinterpret_cast<uint64_t*>(c.ws + size_t(c.rows) * p.splits * 16);
    const size_t smem = c.top ? size_t(kLpCap + kLpMaxSplit) * 8 : 0;
    const unsigned grid = unsigned(c.rows * p.splits);
    const auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (p.U == 8 && c.top) logprobs_kernel<DT, 8, true><<<grid, kLpThreads, smem, s>>>(a);
        else if (p.U == 8) logprobs_kernel<DT, 8, false><<<grid, kLpThreads, smem, s>>>(a);
        else if (c.top) logprobs_kernel<DT, 2, true><<<grid, kLpThreads, smem, s>>>(a);
        else logprobs_kernel<DT, 2, false><<<grid, kLpThreads, smem, s>>>(a);
    };
    if (c.x_dtype == DT_F32) go(std::integral_constant<int, DT_F32>());
    else if (c.x_dtype == DT_F16) go(std::integral_constant<int, DT_F16>());
    else go(std::integral_constant<int, DT_BF16>());
    return cudaGetLastError();
}

}  // namespace exl3
