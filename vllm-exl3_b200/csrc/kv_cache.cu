// kv_cache.cu -- a step's bookkeeping for the paged cache, and the writes into it.
//
// kv_plan: for request b with len_b cached and new_b new tokens and pages of P
//   have_b = ceil(len_b / P), need_b = ceil((len_b + new_b) / P) - have_b,
//   start_b = cursor + sum_{a<b} need_a, cu_b = sum_{a<b} new_a,
//   table[b][have_b + i] = free[start_b + i],  0 <= i < need_b,
//   token t of request b: pos = len_b + t - cu_b, slot = table[b][pos / P] * P + pos % P.
// Every CTA scans the requests (B values, from L2) and then fills its share of
// the tokens and of the table: no second launch, no wait between CTAs.  A
// thread looks its request up in the scanned sums by bisection in shared
// memory.  New pages are read from the free list, not from the table, so the
// table's writers and readers need no order.
//
// kv_append: a run is consecutive tokens at consecutive slots of one page, so it
// ends within its tile.  A CTA takes the runs that START in its window of
// tokens, for one kv head, K and V: every tile has one writer, and its scale is
// settled without a second pass over memory.  A run whose page the kept token
// before it shares (slots that repeat, jump or turn back, a skipped row inside
// a page) would be a second writer: it is skipped with a status.
// Rows are read once, 16 bytes a lane, and stay in registers between the
// maximum and the coding: runs of up to 8 iterations of one warp are a warp's
// alone (no barrier), longer ones the CTA's.  Bound: HBM, 2 bytes read and 1
// written per value.
//
// Measured (launches in a graph): the plan of 64 requests, a token each, 3.6 us,
// of 512 with 23318 tokens 5.3 us: one launch and its chain of reads (lengths,
// scan, bisection, table), the bytes are nothing.  64 tokens of 4 heads, dim
// 128, into pages of 16: 5.5 us, the same kind of chain (slot, run, rows and
// page, scale, codes).  8190 tokens of 8 heads, pages of 64: 13.5 us with rows
// in L2 (3.7 TB/s), 18.5 from HBM as a lone call (2.7 TB/s, 2.4 times its 7.7 us
// at the measured copy rate); a CTA's loads, reduction and stores follow one
// another, and two or three CTAs per SM hide that in part.
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "kv_common.cuh"

namespace exl3 {

constexpr int kPlanThreads = 512;

struct KvPlanArgs {
    const int32_t *lens, *fresh;  // [B]
    int B;
    int32_t* table;  // [B][width]
    int width;
    const int32_t* free_pages;  // [n_free]
    int n_free;
    const int32_t* cursor;
    int shift;  // pages of 1 << shift tokens
    int n_tokens;
    int32_t *kv_lens, *cu, *positions;  // [B], [B + 1], [n_tokens]
    int64_t* slots;                     // [n_tokens]
    int32_t* cursor_out;
    int* status;
};

__device__ __forceinline__ int pages_of(int tokens, int shift) { return int((uint32_t(tokens) + (1u << shift) - 1) >> shift); }

__device__ __forceinline__ int clamp32(long long v) { return int(min(v, (long long)INT32_MAX)); }

// last i in [0, n) with sums[i] <= v; sums[0] = 0 <= v
__device__ __forceinline__ int find_segment(const int32_t* sums, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const KvPlanArgs a) {
    extern __shared__ int32_t plan_smem[];
    int32_t* cu = plan_smem;            // [B + 1] token sums
    int32_t* cp = plan_smem + a.B + 1;  // [B + 1] new-page sums
    __shared__ longlong2 warp_sum[kPlanThreads / 32];
    __shared__ longlong2 carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) carry = make_longlong2(0, 0);
    const int base = *a.cursor;
    bool bad = base < 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int len = 0, n = 0, need = 0;
        if (b < a.B) {
            len = a.lens[b], n = a.fresh[b];
            if (len < 0 || n < 0) bad = true, len = max(len, 0), n = max(n, 0);
            if (n > INT32_MAX - len) bad = true, n = INT32_MAX - len;
            // more than list and table hold changes nothing, and makes no longer loop below
            need = int(min(int64_t(pages_of(len + n, a.shift) - pages_of(len, a.shift)), int64_t(a.n_free) + a.width + 1));
            if (blockIdx.x == 0) a.kv_lens[b] = len + n;
        }
        longlong2 s = make_longlong2(n, need);  // sums of what a caller may have got wrong: they pass 32 bits
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, s.x, d), y = __shfl_up_sync(0xffffffffu, s.y, d);
            if (lane >= d) s.x += x, s.y += y;
        }
        if (lane == 31) warp_sum[warp] = s;
        __syncthreads();
        longlong2 before = carry;
        for (int w = 0; w < warp; ++w) before.x += warp_sum[w].x, before.y += warp_sum[w].y;
        if (b < a.B) cu[b] = clamp32(before.x + s.x - n), cp[b] = clamp32(before.y + s.y - need);
        __syncthreads();
        if (tid == kPlanThreads - 1) carry = make_longlong2(before.x + s.x, before.y + s.y);
        __syncthreads();
    }
    const int total = clamp32(carry.x), pages = clamp32(carry.y);
    if (tid == 0) cu[a.B] = total, cp[a.B] = pages;
    __syncthreads();

    const int i0 = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
    for (int b = i0; b <= a.B; b += step) a.cu[b] = min(cu[b], a.n_tokens);
    for (int64_t p = i0; p < pages; p += step) {
        const int b = find_segment(cp, a.B, int(p));
        const int col = pages_of(max(a.lens[b], 0), a.shift) + int(p) - cp[b];
        const int64_t at = int64_t(base) + p;
        if (at >= a.n_free) bad = true;
        if (col < a.width) a.table[int64_t(b) * a.width + col] = at >= 0 && at < a.n_free ? a.free_pages[at] : -1;
        else bad = true;
    }
    for (int64_t t = i0; t < a.n_tokens; t += step) {
        int pos = 0;
        int64_t slot = -1;
        if (t < total) {
            const int b = find_segment(cu, a.B, int(t));
            const int len = max(a.lens[b], 0);
            pos = len + (int(t) - cu[b]);
            const int col = pos >> a.shift, have = pages_of(len, a.shift);
            int page = -1;
            if (col < a.width) {
                const int64_t at = int64_t(base) + cp[b] + col - have;
                if (col < have) page = a.table[int64_t(b) * a.width + col];
                else if (at >= 0 && at < a.n_free) page = a.free_pages[at];
            }
            if (page >= 0) slot = (int64_t(page) << a.shift) + (pos & ((1 << a.shift) - 1));
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    if (i0 == 0) {
        // pages beyond the list were not handed out
        a.cursor_out[0] = int32_t(max(int64_t(base), min(int64_t(base) + pages, int64_t(a.n_free))));
        if (total > a.n_tokens) bad = true;
    }
    if (bad) set_status(a.status, DEV_BAD_INDEX);
}

int num_sms_cached() {
    static std::atomic<int> sms[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return num_sms_current();
    int n = sms[dev].load(std::memory_order_relaxed);
    if (n == 0) sms[dev].store(n = num_sms_current(), std::memory_order_relaxed);
    return n;
}

cudaError_t run_kv_plan(const KvPlanCall& c, cudaStream_t s) {
    KvPlanArgs a;
    a.lens = c.lens, a.fresh = c.fresh, a.B = c.requests;
    a.table = c.table, a.width = c.width, a.free_pages = c.free_pages, a.n_free = c.n_free, a.cursor = c.cursor;
    a.shift = page_shift(c.page), a.n_tokens = c.n_tokens, a.kv_lens = c.kv_lens, a.cu = c.cu, a.positions = c.positions;
    a.slots = c.slots, a.cursor_out = c.cursor_out, a.status = c.status;
    const size_t smem = size_t(a.B + 1) * 8;
    const int work = c.n_tokens > c.requests ? c.n_tokens : c.requests;
    // two tokens a thread: enough CTAs for the stores, few enough that their scans stay one wave
    int grid = (work + 2 * kPlanThreads - 1) / (2 * kPlanThreads);
    grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = raise_smem(kv_plan_kernel, size_t(kKvMaxRequests + 1) * 8, done);
    if (e != cudaSuccess) return e;
    kv_plan_kernel<<<grid, kPlanThreads, smem, s>>>(a);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------

constexpr int kMaxPage = 128;
constexpr int kAppendHold = 8;  // 16-byte loads of a lane between maximum and coding

struct KvAppendArgs {
    const uint16_t* x[2];   // K and V rows [T][heads][dim] with strides
    int64_t tok_stride[2], head_stride[2];
    const int64_t* slots;   // [T]
    int64_t T;
    uint8_t* cache[2];      // [pages][heads][page][dim]
    float* scale[2];        // [pages][heads]
    int64_t pages;
    int heads, shift;       // pages of 1 << shift tokens
    int window;             // tokens whose runs a CTA takes: at most a page
    int* status;
};

template <bool BF16>
__device__ __forceinline__ float2 pair_to_float(uint32_t v) {
    if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// the larger magnitude of two pairs, NaN if either is
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    a &= 0x7fff7fffu, b &= 0x7fff7fffu;
    if constexpr (BF16) {
        const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    } else {
        const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
}

template <bool E4M3, bool BF16, int D, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) kv_append_kernel(const KvAppendArgs a) {
    constexpr int LPR = D / 8;              // lanes per row (8 values each)
    constexpr int RPW = 32 / LPR;           // rows per warp and iteration; even rows are K's, odd ones V's
    constexpr int kWarps = THREADS / 32;
    constexpr int kAlone = kAppendHold * RPW / 2;  // tokens of a run that one warp holds
    __shared__ int64_t slots_near[3 * kMaxPage];   // of the tokens from a page's length before the window on
    __shared__ uint32_t starts[(2 * kMaxPage) / 32];
    __shared__ int16_t begins[kMaxPage + 1];       // the window's runs: first token
    __shared__ int n_runs;
    __shared__ int amax[2];
    const int sh = a.shift, P = 1 << sh, W = a.window, span = (W + P + 31) & ~31;
    const int h = blockIdx.y;
    const int64_t w0 = int64_t(blockIdx.x) * W;
    const int64_t* slot = slots_near + P;  // slot[i]: of token w0 + i, -1: skipped, -2: before the call
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    for (int i = tid; i < P + span; i += THREADS) {
        const int64_t t = w0 - P + i;
        int64_t v = t >= 0 && t < a.T ? a.slots[t] : -1;
        if (v >= (a.pages << sh)) {
            if (h == 0 && i >= P) set_status(a.status, DEV_BAD_INDEX);
            v = -1;
        }
        slots_near[i] = t < 0 ? -2 : v < 0 ? -1 : v;
    }
    if (tid == 0) n_runs = 0;
    __syncthreads();
    for (int i = tid; i < span; i += THREADS) {
        const int64_t v = slot[i], u = slot[i - 1];
        // skipped tokens count as a run of their own, so that they end the one before
        const bool start = v >= 0 ? v != u + 1 || !(v & (P - 1)) : u >= 0;
        const uint32_t m = __ballot_sync(0xffffffffu, start);
        if (lane == 0) starts[i >> 5] = m;
        if (start && v >= 0 && i < W) {
            int64_t before = u;  // the kept token before this one, up to a page's length back
            for (int j = i - 2; before == -1 && j >= i - P; --j) before = slot[j];
            if (before >= 0 && (before >> sh) == (v >> sh)) {
                if (h == 0) set_status(a.status, DEV_BAD_INDEX);
            } else {
                begins[atomicAdd(&n_runs, 1)] = int16_t(i);  // in any order
            }
        }
    }
    __syncthreads();
    const int last = int(min(int64_t(span), a.T - w0));
    auto run_end = [&](int i) {  // first token after the run that begins at i
        int w = (i + 1) >> 5;
        if (i + 1 >= span) return last;
        uint32_t m = starts[w] & (0xffffffffu << ((i + 1) & 31));
        while (m == 0 && ++w < (span >> 5)) m = starts[w];
        return min(m ? (w << 5) + __ffs(m) - 1 : span, last);
    };

    const int sub = lane / LPR, which = sub & 1, col = (lane % LPR) * 8;
    const uint16_t* x = (which ? a.x[1] + h * a.head_stride[1] : a.x[0] + h * a.head_stride[0]) + col;
    const int64_t ts = which ? a.tok_stride[1] : a.tok_stride[0];
    uint8_t* cache = (which ? a.cache[1] : a.cache[0]) + col;
    float* scales = which ? a.scale[1] : a.scale[0];
    // Rows of tokens first + row / 2 (K where even): this lane's are row0, row0 + step, ...
    uint4 v[kAppendHold];
    // over the lanes of a row, and over the warp's rows of the same kind; NaN if one is
    auto over_lanes = [&](float m) {
        #pragma unroll
        for (int d = 1; d < LPR; d <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
        return RPW == 4 ? max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2 * LPR)) : m;
    };
    auto load = [&](int first, int n, int row0, int step) {  // and their largest magnitude
        #pragma unroll
        for (int i = 0; i < kAppendHold; ++i) {
            const int t = (row0 + i * step) >> 1;
            v[i] = t < n ? __ldg(reinterpret_cast<const uint4*>(x + (w0 + first + t) * ts)) : make_uint4(0, 0, 0, 0);
        }
        uint32_t m = 0;
        #pragma unroll
        for (int i = 0; i < kAppendHold; ++i)
            m = max_abs2<BF16>(m, max_abs2<BF16>(max_abs2<BF16>(v[i].x, v[i].y), max_abs2<BF16>(v[i].z, v[i].w)));
        const float2 f = pair_to_float<BF16>(m);
        return over_lanes(max_nan(fabsf(f.x), fabsf(f.y)));
    };
    auto largest_number = [&]() {  // of rows with NaN in them
        float m = 0.f;
        #pragma unroll
        for (int i = 0; i < kAppendHold; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            #pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float2 f = pair_to_float<BF16>(w[q]);
                m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));  // fmaxf leaves NaN out
            }
        }
        return over_lanes(m);
    };
    // ODD: there may be NaN, or numbers beyond what the largest scale brings into the codes' range
    auto code = [&](auto odd, int first, int n, int row0, int step, int e) {
        constexpr bool ODD = decltype(odd)::value;
        const float inv = exp2_int(-e);
        const int64_t s = slot[first];
        const int64_t base = (((s >> sh) * a.heads + h) << sh) + (s & (P - 1));
        #pragma unroll
        for (int i = 0; i < kAppendHold; ++i) {
            const int t = (row0 + i * step) >> 1;
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            float f[8];
            #pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float2 p = pair_to_float<BF16>(w[q]);
                f[2 * q] = p.x * inv, f[2 * q + 1] = p.y * inv;
            }
            uint2 c;
            if constexpr (!ODD && !E4M3) {
                // x / s + 1.5 * 2^23 has the rounded code in its low byte
                uint32_t b[8];
                #pragma unroll
                for (int q = 0; q < 8; ++q) b[q] = __float_as_uint(f[q] + 12582912.f);
                c.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
                c.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
            } else {
                if constexpr (ODD && E4M3) {
                    // A NaN of V goes into the token's key instead: every row that sees the token becomes
                    // NaN, and no other (0 * NaN would reach those that do not).
                    bool nan = false;
                    #pragma unroll
                    for (int q = 0; q < 8; ++q) nan |= f[q] != f[q];
                    uint32_t bad = __ballot_sync(0xffffffffu, nan && which);
                    bad = (bad >> ((sub | 1) * LPR)) & ((1u << LPR) - 1u);
                    if (bad) {
                        #pragma unroll
                        for (int q = 0; q < 8; ++q) f[q] = which ? (f[q] == f[q] ? f[q] : 0.f) : NAN;
                    }
                }
                c.x = encode4<E4M3>(f[0], f[1], f[2], f[3]), c.y = encode4<E4M3>(f[4], f[5], f[6], f[7]);
            }
            if (t < n) *reinterpret_cast<uint2*>(cache + (base + t) * D) = c;
        }
    };
    constexpr float kMost = (E4M3 ? 448.f : 127.f) * 1099511627776.f;  // at the largest scale, 2^40
    // the scale of the run's tile, and the one it had
    auto settle = [&](int first, float m, int& old) {
        const int64_t s = slot[first];
        const float* sc = scales + (s >> sh) * a.heads + h;
        int e = scale_exponent<E4M3>(m);
        old = e;
        if (s & (P - 1)) {  // joins a page that holds tokens already
            old = stored_exponent(*sc);
            e = max(e, old);
        }
        return e;
    };
    auto publish = [&](int first, int e) {
        const int64_t s = slot[first];
        scales[(s >> sh) * a.heads + h] = exp2_int(e);
    };
    // the scale grew: the tile's older codes (rows row0, row0 + step, ... of its first tokens) move to it
    auto again = [&](int first, int row0, int step, int old, int e) {
        const int64_t s = slot[first], base = ((s >> sh) * a.heads + h) << sh;
        const int off = int(s & (P - 1));
        const float f = exp2_int(max(old - e, -126));
        for (int r = row0; (r >> 1) < off; r += step) {
            uint2* p = reinterpret_cast<uint2*>(cache + (base + (r >> 1)) * D);
            const uint2 c = *p;
            float u[4], w[4];
            decode4<E4M3>(c.x, u);
            decode4<E4M3>(c.y, w);
            *p = make_uint2(encode4<E4M3>(u[0] * f, u[1] * f, u[2] * f, u[3] * f),
                            encode4<E4M3>(w[0] * f, w[1] * f, w[2] * f, w[3] * f));
        }
    };

    bool longs = false;
    for (int k = warp; k < n_runs; k += kWarps) {
        const int first = begins[k], n = run_end(first) - first;
        if (n > kAlone) {
            longs = true;
            continue;
        }
        float m = load(first, n, sub, RPW);
        const bool odd = __any_sync(0xffffffffu, !(m <= kMost));
        if (odd) m = largest_number();
        int old;
        const int e = settle(first, m, old);
        __syncwarp();
        if (lane % LPR == 0 && sub < 2) publish(first, e);
        if (odd) code(std::true_type(), first, n, sub, RPW, e);
        else code(std::false_type(), first, n, sub, RPW, e);
        if (old < e) again(first, sub, RPW, old, e);
    }
    if (!__syncthreads_or(longs)) return;
    for (int k = 0; k < n_runs; ++k) {
        const int first = begins[k], n = run_end(first) - first;
        if (n <= kAlone) continue;
        if (tid < 2) amax[tid] = 0;
        __syncthreads();
        const float m = load(first, n, warp * RPW + sub, kWarps * RPW);
        if (lane % LPR == 0 && sub < 2) atomicMax(&amax[which], __float_as_int(m));  // of floats >= 0; NaN is the largest
        __syncthreads();
        const bool odd = !(__int_as_float(amax[0]) <= kMost && __int_as_float(amax[1]) <= kMost);
        if (odd) {
            const float number = largest_number();
            __syncthreads();
            if (tid < 2) amax[tid] = 0;
            __syncthreads();
            if (lane % LPR == 0 && sub < 2) atomicMax(&amax[which], __float_as_int(number));
            __syncthreads();
        }
        int old;
        const int e = settle(first, __int_as_float(amax[which]), old);
        __syncthreads();  // all have read the old scale
        if (warp == 0 && lane % LPR == 0 && sub < 2) publish(first, e);
        if (odd) code(std::true_type(), first, n, warp * RPW + sub, kWarps * RPW, e);
        else code(std::false_type(), first, n, warp * RPW + sub, kWarps * RPW, e);
        if (old < e) again(first, warp * RPW + sub, kWarps * RPW, old, e);
    }
}

template <bool E4M3, bool BF16, int D>
static void launch_append(const KvAppendArgs& a, dim3 grid, cudaStream_t s) {
    // a page's rows of K and V fit the CTA's registers: 2 P D / 8 lanes' worth in kAppendHold iterations
    if (a.shift == 7) kv_append_kernel<E4M3, BF16, D, 512><<<grid, 512, 0, s>>>(a);
    else kv_append_kernel<E4M3, BF16, D, 256><<<grid, 256, 0, s>>>(a);
}

cudaError_t run_kv_append(const KvAppendCall& c, int sms, cudaStream_t s) {
    if (c.tokens <= 0) return cudaSuccess;
    KvAppendArgs a;
    for (int i = 0; i < 2; ++i) {
        a.x[i] = static_cast<const uint16_t*>(c.x[i]), a.tok_stride[i] = c.tok_stride[i], a.head_stride[i] = c.head_stride[i];
        a.cache[i] = static_cast<uint8_t*>(c.cache[i]), a.scale[i] = c.scale[i];
    }
    a.slots = c.slots, a.T = c.tokens, a.pages = c.pages, a.heads = c.heads, a.shift = page_shift(c.page), a.status = c.status;
    // Windows of a page where that gives every SM a CTA, else of 16 tokens.  us with 16 / a page (8 heads,
    // pages of 64): 64 single tokens 5.2 / 14.1, 512 6.6 / 14.5, a prompt of 2000 7.7 / 6.5, of 4000 11.3 / 8.1
    a.window = (c.tokens / c.page) * c.heads >= sms ? c.page : 16;
    const dim3 grid(unsigned((c.tokens + a.window - 1) / a.window), unsigned(c.heads), 1);
    const auto by_dim = [&](auto e4, auto bf) {
        constexpr bool E = decltype(e4)::value, B = decltype(bf)::value;
        c.dim == 128 ? launch_append<E, B, 128>(a, grid, s) : launch_append<E, B, 64>(a, grid, s);
    };
    const bool bf16 = c.x_dtype == DT_BF16;
    if (c.e4m3) bf16 ? by_dim(std::true_type(), std::true_type()) : by_dim(std::true_type(), std::false_type());
    else bf16 ? by_dim(std::false_type(), std::true_type()) : by_dim(std::false_type(), std::false_type());
    return cudaGetLastError();
}

}  // namespace exl3
