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
// kv_append: one CTA per (window of P tokens, kv head, K or V); it owns the
// runs (consecutive tokens of one page) that START in its window, so every
// tile has one writer and its scale can be settled in shared memory: rows are
// read once from HBM for the run's largest magnitude and once more, from L1,
// to be coded.
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

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
    __shared__ int2 warp_sum[kPlanThreads / 32];
    __shared__ int2 carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) carry = make_int2(0, 0);
    const int base = *a.cursor;
    bool bad = base < 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        int len = 0, n = 0, need = 0;
        if (b < a.B) {
            len = a.lens[b], n = a.fresh[b];
            if (len < 0 || n < 0) bad = true, len = max(len, 0), n = max(n, 0);
            need = pages_of(len + n, a.shift) - pages_of(len, a.shift);
            if (blockIdx.x == 0) a.kv_lens[b] = len + n;
        }
        int2 s = make_int2(n, need);
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, s.x, d), y = __shfl_up_sync(0xffffffffu, s.y, d);
            if (lane >= d) s.x += x, s.y += y;
        }
        if (lane == 31) warp_sum[warp] = s;
        __syncthreads();
        int2 before = carry;
        for (int w = 0; w < warp; ++w) before.x += warp_sum[w].x, before.y += warp_sum[w].y;
        if (b < a.B) cu[b] = before.x + s.x - n, cp[b] = before.y + s.y - need;
        __syncthreads();
        if (tid == kPlanThreads - 1) carry = make_int2(before.x + s.x, before.y + s.y);
        __syncthreads();
    }
    const int total = carry.x, pages = carry.y;
    if (tid == 0) cu[a.B] = total, cp[a.B] = pages;
    __syncthreads();

    const int i0 = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
    for (int b = i0; b <= a.B; b += step) a.cu[b] = min(cu[b], a.n_tokens);
    for (int p = i0; p < pages; p += step) {
        const int b = find_segment(cp, a.B, p);
        const int col = pages_of(max(a.lens[b], 0), a.shift) + p - cp[b];
        const int64_t at = int64_t(base) + p;
        if (at >= a.n_free) bad = true;
        if (col < a.width) a.table[int64_t(b) * a.width + col] = at >= 0 && at < a.n_free ? a.free_pages[at] : -1;
        else bad = true;
    }
    for (int t = i0; t < a.n_tokens; t += step) {
        int pos = 0;
        int64_t slot = -1;
        if (t < total) {
            const int b = find_segment(cu, a.B, t);
            const int len = max(a.lens[b], 0);
            pos = len + t - cu[b];
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
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (e != cudaSuccess) return e;
    }
    kv_plan_kernel<<<grid, kPlanThreads, smem, s>>>(a);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------

constexpr int kAppendThreads = 256;
constexpr int kMaxPage = 128;

struct KvAppendArgs {
    const void* x[2];       // K and V rows [T][heads][dim] with strides
    int64_t tok_stride[2], head_stride[2];
    const int64_t* slots;   // [T]
    int64_t T;
    uint8_t* cache[2];      // [pages][heads][page][dim]
    float* scale[2];        // [pages][heads]
    int64_t pages;
    int heads, shift;  // pages of 1 << shift tokens
    int* status;
};

template <bool BF16>
__device__ __forceinline__ float2 pair_to_float(uint32_t v) {
    if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const KvAppendArgs a) {
    // indices into the window's arrays: 0 is the token before the window
    __shared__ int64_t slot[2 * kMaxPage + 1];
    __shared__ uint32_t starts[(2 * kMaxPage) / 32];  // bit i: token w0 + i begins a run
    __shared__ int amax[kMaxPage];                    // of the run that begins at token w0 + i (bits of a float >= 0)
    __shared__ int exps[kMaxPage], olds[kMaxPage];
    const int sh = a.shift, P = 1 << sh, W = 2 * P;
    const int h = blockIdx.y, which = blockIdx.z;
    const int64_t w0 = int64_t(blockIdx.x) * P;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kAppendThreads / 32;

    for (int i = tid; i <= W; i += kAppendThreads) {
        const int64_t t = w0 - 1 + i;
        int64_t v = t >= 0 && t < a.T ? a.slots[t] : -1;
        if (v >= (a.pages << sh)) {
            if (h == 0 && which == 0 && i > 0) set_status(a.status, DEV_BAD_INDEX);
            v = -1;
        }
        slot[i] = v < 0 ? -1 : v;
    }
    if (tid < P) amax[tid] = 0;
    __syncthreads();
    for (int i = tid; i < W; i += kAppendThreads) {
        const int64_t v = slot[i + 1], u = slot[i];
        const bool start = v >= 0 ? u < 0 || (u >> sh) != (v >> sh) : u >= 0;  // a run of skipped tokens counts as one
        const uint32_t m = __ballot_sync(0xffffffffu, start || (i == 0 && v < 0));
        if (lane == 0) starts[i >> 5] = m;
    }
    __syncthreads();
    // first token of token i's run, -1 if it lies before the window or the token is skipped
    auto run_of = [&](int i) {
        if (slot[i + 1] < 0) return -1;
        int w = i >> 5;
        uint32_t m = starts[w] & (0xffffffffu >> (31 - (i & 31)));
        while (m == 0 && w > 0) m = starts[--w];
        return m ? (w << 5) + 31 - __clz(m) : -1;
    };
    const uint16_t* x = static_cast<const uint16_t*>(a.x[which]) + h * a.head_stride[which];
    const int64_t ts = a.tok_stride[which];
    const int last = int(min(int64_t(W), a.T - w0));
    constexpr int V = D / 32;  // values per lane: 4 or 2

    auto row = [&](int i, float (&v)[V]) {
        const uint16_t* p = x + (w0 + i) * ts + lane * V;
        if constexpr (V == 4) {
            const uint2 r = *reinterpret_cast<const uint2*>(p);
            const float2 lo = pair_to_float<BF16>(r.x), hi = pair_to_float<BF16>(r.y);
            v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
        } else {
            const float2 lo = pair_to_float<BF16>(*reinterpret_cast<const uint32_t*>(p));
            v[0] = lo.x, v[1] = lo.y;
        }
    };
    for (int i = warp; i < last; i += kWarps) {
        const int r = run_of(i);
        if (r >= P) break;   // this run and what follows belong to later windows
        if (r < 0) continue;
        float v[V], m = 0.f;
        row(i, v);
        #pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, fabsf(v[j]));  // fmaxf leaves NaN out
        const int mi = __reduce_max_sync(0xffffffffu, __float_as_int(m));
        if (lane == 0) atomicMax(&amax[r], mi);
    }
    __syncthreads();
    if (tid < P && tid < last && run_of(tid) == tid) {
        const int64_t v = slot[tid + 1], page = v >> sh;
        float* sc = a.scale[which] + page * a.heads + h;
        int e = scale_exponent<E4M3>(__int_as_float(amax[tid])), old = e;
        if (v & (P - 1)) {  // joins a page that holds tokens already
            old = stored_exponent(*sc);
            e = max(e, old);
        }
        exps[tid] = e, olds[tid] = old;
        *sc = exp2_int(e);
    }
    __syncthreads();
    auto store = [&](int64_t at, const float (&v)[V]) {
        uint8_t* p = a.cache[which] + at * D + lane * V;
        if constexpr (V == 4) *reinterpret_cast<uint32_t*>(p) = encode4<E4M3>(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint16_t*>(p) = uint16_t(encode4<E4M3>(v[0], v[1], 0.f, 0.f));
    };
    for (int i = warp; i < last; i += kWarps) {
        const int r = run_of(i);
        if (r >= P) break;
        if (r < 0) continue;
        float v[V];
        row(i, v);
        const float inv = exp2_int(-exps[r]);
        #pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= inv;
        const int64_t s = slot[i + 1];
        const int64_t tile = (((s >> sh) * a.heads + h) << sh);
        const int off = int(s & (P - 1));
        store(tile + off, v);
        if (r != i || olds[r] >= exps[r]) continue;
        // the scale grew: the tile's older codes move to it
        const float f = exp2_int(max(olds[r] - exps[r], -126));
        for (int o = 0; o < off; ++o) {
            const uint8_t* p = a.cache[which] + (tile + o) * D + lane * V;
            const uint32_t w = V == 4 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
            float c[4], u[V];
            decode4<E4M3>(w, c);
            #pragma unroll
            for (int j = 0; j < V; ++j) u[j] = c[j] * f;
            store(tile + o, u);
        }
    }
}

cudaError_t run_kv_append(const KvAppendCall& c, cudaStream_t s) {
    if (c.tokens <= 0) return cudaSuccess;
    KvAppendArgs a;
    for (int i = 0; i < 2; ++i) {
        a.x[i] = c.x[i], a.tok_stride[i] = c.tok_stride[i], a.head_stride[i] = c.head_stride[i];
        a.cache[i] = static_cast<uint8_t*>(c.cache[i]), a.scale[i] = c.scale[i];
    }
    a.slots = c.slots, a.T = c.tokens, a.pages = c.pages, a.heads = c.heads, a.shift = page_shift(c.page), a.status = c.status;
    const dim3 grid(unsigned((c.tokens + c.page - 1) / c.page), unsigned(c.heads), 2);
    const auto go = [&](auto e4m3, auto bf16, auto dim) {
        kv_append_kernel<decltype(e4m3)::value, decltype(bf16)::value, decltype(dim)::value>
            <<<grid, kAppendThreads, 0, s>>>(a);
    };
    const auto by_dim = [&](auto e4m3, auto bf16) {
        if (c.dim == 128) go(e4m3, bf16, std::integral_constant<int, 128>());
        else go(e4m3, bf16, std::integral_constant<int, 64>());
    };
    const bool bf16 = c.x_dtype == DT_BF16;
    if (c.e4m3) bf16 ? by_dim(std::true_type(), std::true_type()) : by_dim(std::true_type(), std::false_type());
    else bf16 ? by_dim(std::false_type(), std::true_type()) : by_dim(std::false_type(), std::false_type());
    return cudaGetLastError();
}

}  // namespace exl3
