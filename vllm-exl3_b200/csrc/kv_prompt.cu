// kv_prompt.cu -- attention over the paged 8-bit cache, many query rows per request.
//
// The mathematics of kv_attend.cu (weights 2^(s + log2 vscale - m), codes into
// the tensor core as they are), with 256 query rows per CTA instead of 8 or
// 16: a row is one (token, query head) of the kv head's group, so a tile's
// rows share the keys.  Bound: the tensor core, 4 D flops per (row, key); the
// exponential unit comes as close (128 x 128 weights take 1024 clocks of one
// and, with D = 128, 1024 of the other).
//
// Two 128-row tiles per CTA, so that one's products run while the other's
// weights are computed.  13 warps:
//   0-3, 4-7  one row per thread: running maximum, weights, sums (tiles 0 and 1)
//   8-11      codes of 128 keys from global memory to f16 in shared memory
//             (128-byte swizzle; K is a K-major operand, V an MN-major one: the same bytes)
//   12        one thread issues S = Q K^T and O += P V (tcgen05, fp32 in TMEM)
// TMEM: S0 S1 (128 columns each; the weights, f16, take the place of the
// scores that they came from and are the A operand of P V), O0 O1.
// The order of the issue S0 S1 | PV0 S0' PV1 S1' | ... keeps one tile's
// products behind the other's weights; tcgen05 runs one thread's products in order.
//
// O is rescaled only when a row's maximum grows by more than 2^8 over the
// reference its weights are taken against: until then weights up to 2^8 (f16
// holds them, the sums are fp32) cost nothing, and the final division is by a
// sum over the same reference.
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "kv_attend.cuh"
#include "tc_common.cuh"

namespace exl3 {

constexpr int kPrThreads = 13 * 32;
constexpr int kPrKeys = 128;        // keys per step
constexpr int kPrRows = 256;        // query rows per CTA
constexpr int kPrScaleSlots = 4;
constexpr float kPrSlack = 8.f;     // log2: growth of the maximum that is let pass
constexpr uint32_t kPrTmem = 512;

struct PrSmem {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], sc_full[kPrScaleSlots];
    uint32_t tmem;
    int abort_flag, last;
    int64_t scan[13];
    int found_b;
    int64_t found_base;
    float4 sc[kPrScaleSlots][8];  // of 16 keys: K scale, log2 V scale, 1 / V scale, 1 if the page exists
    float wt[kPrRows];
};

template <int D>
constexpr size_t pr_smem_bytes() {
    return 1024 + size_t(kPrRows) * D * 2 + 4 * size_t(kPrKeys) * D * 2 + sizeof(PrSmem);
}

__device__ __forceinline__ bool pr_wait(uint64_t* bar, uint32_t parity, int* status, volatile int* abort_flag) {
    if (*abort_flag) return false;
    if (mbar_wait(bar, parity, status)) return true;
    *abort_flag = 1;
    return false;
}

// MN-major operand, 128-byte swizzle: 64-element (128-byte) rows along MN, one
// per k; 8 k to an atom (SBO 1024); the next 64 of MN are `lbo` bytes on.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= uint64_t((smem_addr >> 4) & 0x3FFF);
    d |= uint64_t(lbo >> 4) << 16;
    d |= uint64_t(1024 >> 4) << 32;
    d |= uint64_t(1) << 46;
    d |= uint64_t(2) << 61;
    return d;
}

// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}

__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load_wait(uint32_t (&r)[32]) {
    // the registers are operands, so that nothing reads them before the wait
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

struct PrArgs {
    KvAttendArgs a;
    int splits;  // parts of a tile's keys (at most; no more than its steps)
};

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(kPrThreads, 1) kv_prompt_kernel(const PrArgs args) {
    constexpr int kBlk = kPrKeys * 128;        // bytes of a 64-dim block of 128 rows
    constexpr int kTile = (D / 64) * kBlk;     // a 128-row f16 tile
    const KvAttendArgs& a = args.a;
    extern __shared__ char pr_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(pr_raw) + 1023) & ~uintptr_t(1023));
    char* vst = smem;              // 2 stages
    char* kst = vst + 2 * kTile;   // 2 stages
    char* qs = kst + 2 * kTile;    // 2 tiles
    PrSmem& sm = *reinterpret_cast<PrSmem*>(qs + 2 * kTile);
    volatile int* abort_flag = &sm.abort_flag;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int Hk = a.kv_heads, G = a.group, P = 1 << a.shift;

    // --- which tile ---
    auto tiles_of = [&](int b) {
        const int64_t cols = int64_t(a.cu ? max(a.cu[b + 1] - a.cu[b], 0) : 1) * G;
        return cols > a.few ? (cols + kPrRows - 1) / kPrRows : int64_t(0);
    };
    const int64_t item = blockIdx.x / args.splits;
    const int split = int(blockIdx.x % args.splits);
    int b = 0;
    int64_t tile = item / Hk;
    const int hk = int(item % Hk);
    {
        const int per = (a.requests + kPrThreads - 1) / kPrThreads;
        int64_t mine = 0;
        for (int i = 0; i < per; ++i)
            if (tid * per + i < a.requests) mine += tiles_of(tid * per + i);
        int64_t incl = mine;
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) sm.scan[warp] = incl;
        __syncthreads();
        int64_t total = 0;
        for (int w = 0; w < kPrThreads / 32; ++w) {
            if (w == warp) incl += total;
            total += sm.scan[w];
        }
        if (tile >= total) return;  // the grid covers the most tiles there could be
        tile = total - 1 - tile;    // a request's last rows, whose keys are the most, first
        if (tile >= incl - mine && tile < incl) {
            int64_t base = incl - mine;
            int i = tid * per;
            for (int64_t n; tile >= base + (n = tiles_of(i)); ++i) base += n;
            sm.found_b = i, sm.found_base = base;
        }
        __syncthreads();
        b = sm.found_b;
        tile -= sm.found_base;
    }
    const int64_t row0 = a.cu ? a.cu[b] : b;
    const int fresh = a.cu ? a.cu[b + 1] - int(row0) : 1;
    const int len = int(min(int64_t(max(a.kv_lens[b], 0)), int64_t(a.width) << a.shift));
    const int64_t col0 = tile * kPrRows;
    const int rows = int(min(int64_t(fresh) * G - col0, int64_t(kPrRows)));
    const int nt = rows > 128 ? 2 : 1;
    // keys that any row of the tile sees
    const int pos_first = len - fresh + int(col0 / G), pos_last = len - fresh + int((col0 + rows - 1) / G);
    const int hi_all = max(min(pos_last + 1, len), 0);
    const int lo_all = a.window > 0 ? max(pos_first + 1 - a.window, 0) : 0;
    const int k_begin = min(lo_all, hi_all) & ~(kPrKeys - 1);
    const int steps_all = (hi_all - k_begin + kPrKeys - 1) / kPrKeys;
    const int ns = max(min(args.splits, steps_all), 1);
    if (split >= ns) return;
    const int step0 = int(int64_t(steps_all) * split / ns);
    const int steps = int(int64_t(steps_all) * (split + 1) / ns) - step0;
    const int key0 = k_begin + step0 * kPrKeys;

    if (tid == 0) {
        mbar_init(&sm.q_full, 128 * nt);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.k_full[i], 4);
            mbar_init(&sm.v_full[i], 4);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.o_full[i], 1);
            mbar_init(&sm.p_full[i], 128);
        }
        for (int i = 0; i < kPrScaleSlots; ++i) mbar_init(&sm.sc_full[i], 1);
        sm.abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 12) tmem_alloc(&sm.tmem, kPrTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sm.tmem;
    // columns: S0 0, S1 128, O0 256, O1 384
    if (warp < 8) {
        const int t = warp >> 2;
        if (t < nt) {
            // --- this thread's row ---
            const int r = tid & 127, f = t * 128 + r;
            const uint32_t lane_base = uint32_t(32 * (warp & 3)) << 16;
            const uint32_t ts = tm + lane_base + uint32_t(128 * t), to = tm + lane_base + uint32_t(256 + 128 * t);
            const int64_t fc = col0 + f, row = row0 + fc / G;
            const bool live = f < rows && row < a.q_rows;
            float cfac = fabsf(a.scale_log2);
            {
                const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;  // group maxima below need a factor >= 0
                const uint4* qp = reinterpret_cast<const uint4*>(a.q + (live ? row * a.q_tok + int64_t(hk * G + fc % G) * a.q_head : 0));
                uint4 w[D / 8];
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) w[i] = live ? __ldg(qp + i) : make_uint4(0, 0, 0, 0);
                float mul = sign;
                if constexpr (BF16) {
                    // to f16 by a power of two per row: largest magnitude in [2^14, 2^15), so that
                    // values down to 2^-31 of it keep all 8 bits
                    uint32_t m2 = 0;
                    #pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t x = __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu),
                                                    __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
                        m2 = __vmaxu2(m2, x);
                    }
                    const float amax = fmaxf(__uint_as_float(m2 << 16), __uint_as_float(m2 & 0xffff0000u));
                    const int e = min(max((__float_as_int(amax) >> 23) - 127, -100), 100);
                    mul *= exp2_int(14 - e);
                    cfac *= exp2_int(e - 14);
                }
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    auto conv = [&](uint32_t v) {
                        if constexpr (BF16)
                            return pack_half2(__uint_as_float(v << 16) * mul, __uint_as_float(v & 0xffff0000u) * mul);
                        else
                            return sign < 0.f ? v ^ 0x80008000u : v;
                    };
                    const uint4 o = make_uint4(conv(w[i].x), conv(w[i].y), conv(w[i].z), conv(w[i].w));
                    *reinterpret_cast<uint4*>(qs + t * kTile + (i >> 3) * kBlk + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = o;
                }
                fence_async_smem();
                mbar_arrive(&sm.q_full);
            }
            const int pos = len - fresh + int(fc / G);
            const int hi = f < rows ? min(pos + 1, len) : 0;
            const int lo = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
            float ref = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < steps; ++j) {
                const int base = key0 + j * kPrKeys;
                ok = pr_wait(&sm.sc_full[j & 3], (j >> 2) & 1, a.status, abort_flag) &&
                     pr_wait(&sm.s_full[t], j & 1, a.status, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const float4* sc = sm.sc[j & 3];
                bool dead = f < rows && (base + kPrKeys > hi || base < lo);  // rows past the tile's end see nothing and give nothing
                #pragma unroll
                for (int g = 0; g < 8; ++g) dead |= sc[g].w == 0.f;
                const bool edge = __any_sync(0xffffffffu, dead);

                // largest score of the row
                float mx = -INFINITY;
                #pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t v[32];
                    tmem_load32(ts + 32 * h, v);
                    tmem_load_wait(v);
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 s4 = sc[2 * h + g];
                        const int kb = base + 32 * h + 16 * g;
                        float gm = -INFINITY;
                        if (!edge) {
                            #pragma unroll
                            for (int i = 0; i < 16; ++i) gm = fmaxf(gm, __uint_as_float(v[16 * g + i]));
                        } else {
                            #pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (kb + i < hi && kb + i >= lo) gm = fmaxf(gm, __uint_as_float(v[16 * g + i]));
                            if (s4.w == 0.f) gm = -INFINITY;
                        }
                        mx = fmaxf(mx, fmaf(gm, cfac * s4.x, s4.y));
                    }
                }
                if (__any_sync(0xffffffffu, mx > ref + kPrSlack || (ref == -INFINITY && mx > ref))) {
                    const float nref = fmaxf(ref, mx);
                    const float alpha = ref == -INFINITY ? 0.f : ex2(ref - nref);
                    l = ref == nref ? l : l * alpha;
                    const float scale = ref == nref ? 1.f : alpha;
                    ref = nref;
                    if (j > 0) {
                        ok = __all_sync(0xffffffffu, pr_wait(&sm.o_full[t], (j - 1) & 1, a.status, abort_flag));
                        if (!ok) break;
                        tc_fence_after();
                        #pragma unroll 1
                        for (int h = 0; h < D / 32; ++h) {
                            uint32_t o[32];
                            tmem_load32(to + 32 * h, o);
                            tmem_load_wait(o);
                            #pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale);
                            tmem_store32(to + 32 * h, o);
                        }
                    }
                }
                const float off = ref == -INFINITY ? 0.f : ref;
                // weights
                #pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t v[32], p[16];
                    tmem_load32(ts + 32 * h, v);
                    tmem_load_wait(v);
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 s4 = sc[2 * h + g];
                        const int kb = base + 32 * h + 16 * g;
                        const float mul = cfac * s4.x, add = s4.y - off;
                        float sum = 0.f;
                        #pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float x = fmaf(__uint_as_float(v[16 * g + i]), mul, add);
                            float y = fmaf(__uint_as_float(v[16 * g + i + 1]), mul, add);
                            if (edge) {
                                if (kb + i >= hi || kb + i < lo || s4.w == 0.f) x = -INFINITY;
                                if (kb + i + 1 >= hi || kb + i + 1 < lo || s4.w == 0.f) y = -INFINITY;
                            }
                            x = ex2(x), y = ex2(y);
                            sum += x + y;
                            p[8 * g + i / 2] = pack_half2(x, y);
                        }
                        l = fmaf(sum, s4.z, l);
                    }
                    tmem_store16(ts + 16 * h, p);
                }
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(&sm.p_full[t]);
            }
            // --- the row's result ---
            if (steps > 0 && ok) ok = __all_sync(0xffffffffu, pr_wait(&sm.o_full[t], (steps - 1) & 1, a.status, abort_flag));
            tc_fence_after();
            if (ok && ns == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
                const int64_t at = row * a.heads + hk * G + fc % G;
                #pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t o[32];
                    if (steps > 0) {
                        tmem_load32(to + 32 * h, o);
                        tmem_load_wait(o);
                    } else {
                        #pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0u;
                    }
                    uint32_t w[16];
                    #pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float x = __uint_as_float(o[2 * i]) * inv, y = __uint_as_float(o[2 * i + 1]) * inv;
                        if constexpr (BF16) {
                            const __nv_bfloat162 q2 = __floats2bfloat162_rn(x, y);
                            w[i] = *reinterpret_cast<const uint32_t*>(&q2);
                        } else {
                            w[i] = pack_half2(x, y);
                        }
                        if (l == 0.f) w[i] = 0u;
                    }
                    if (live) {
                        uint4* dst = reinterpret_cast<uint4*>(a.out + at * D + 32 * h);
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    }
                }
                if (live && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
            } else if (ok) {
                // partial: [item][split] of {reference, sum} per row, then O rows
                float* part = a.part + (item * args.splits + split) * int64_t(kPrRows) * (D + 2);
                __stcg(part + f, ref);
                __stcg(part + kPrRows + f, l);
                #pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t o[32];
                    tmem_load32(to + 32 * h, o);
                    tmem_load_wait(o);
                    float4* dst = reinterpret_cast<float4*>(part + 2 * kPrRows + f * D + 32 * h);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        __stcg(dst + i, make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                    __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])));
                }
            }
            tc_fence_before();
        }
    } else if (warp < 12) {
        // --- codes to f16 ---
        constexpr int CH = D / 16;           // 16-byte loads per key
        constexpr int RPP = 128 / CH;        // keys per pass
        constexpr int NP = kPrKeys / RPP;
        const int ct = tid - 256, kr = ct / CH, ch = ct % CH;
        const int32_t* row_table = a.table + int64_t(b) * a.width;
        auto page_of = [&](int key) {  // of a key below len
            const int p = row_table[key >> a.shift];
            if (p >= 0 && p < a.pages) return p;
            set_status(a.status, DEV_BAD_INDEX);
            return -1;
        };
        auto pages = [&](int j, int (&pg)[NP]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int key = key0 + j * kPrKeys + i * RPP + kr;
                // keys that no row sees are zeros: their codes may be NaN, and 0 * NaN is not 0
                pg[i] = j < steps && key >= lo_all && key < hi_all ? page_of(key) : -1;
            }
        };
        auto load = [&](const uint8_t* codes, int j, const int (&pg)[NP], uint4 (&w)[NP]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int key = key0 + j * kPrKeys + i * RPP + kr;
                const uint8_t* p = codes + (((int64_t(max(pg[i], 0)) * Hk + hk) << a.shift) + (key & (P - 1))) * D + ch * 16;
                w[i] = pg[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
            }
        };
        auto put = [&](char* dst, const uint4 (&w)[NP], const int (&pg)[NP]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int key = i * RPP + kr;
                const uint32_t in[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                uint32_t o[8];
                #pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t c = code_word<E4M3>(in[q]);
                    o[2 * q] = half2_lo<E4M3>(c), o[2 * q + 1] = half2_hi<E4M3>(c);
                    if (!E4M3 && pg[i] < 0) o[2 * q] = o[2 * q + 1] = 0u;
                }
                // lanes of dims 64 and up store their halves in the other order: 8 lanes, 8 banks of 16 bytes
                char* rowp = dst + (ch >> 2) * kBlk + key * 128;
                const int c0 = 2 * (ch & 3), sw = key & 7;
                const bool flip = ch >= 4;
                const uint4 x = make_uint4(o[0], o[1], o[2], o[3]), y = make_uint4(o[4], o[5], o[6], o[7]);
                *reinterpret_cast<uint4*>(rowp + (((c0 + (flip ? 1 : 0)) ^ sw) << 4)) = flip ? y : x;
                *reinterpret_cast<uint4*>(rowp + (((c0 + (flip ? 0 : 1)) ^ sw) << 4)) = flip ? x : y;
            }
            fence_async_smem();
            __syncwarp();
        };
        auto scales = [&](int j) {  // of 16 keys, by the first 8 threads
            const int key = key0 + j * kPrKeys + 16 * ct;
            if (ct >= 8 || j >= steps || key + 16 <= lo_all || key >= hi_all) return make_float4(0.f, 0.f, 1.f, 1.f);
            const int pg = page_of(key);
            if (pg < 0) return make_float4(0.f, 0.f, 1.f, 0.f);
            const int64_t at = int64_t(pg) * Hk + hk;
            const int ve = stored_exponent(__ldg(a.v_scale + at));
            return make_float4(__ldg(a.k_scale + at), float(ve), exp2_int(-ve), 1.f);
        };
        int pg[NP], pn[NP];
        uint4 kw[NP], vw[NP];
        pages(0, pg);
        load(a.k, 0, pg, kw);
        float4 sc = scales(0);
        bool ok = true;
        for (int j = 0; j < steps; ++j) {
            const int s = j & 1;
            load(a.v, j, pg, vw);
            pages(j + 1, pn);
            if (j >= 2) ok = pr_wait(&sm.k_empty[s], ((j >> 1) - 1) & 1, a.status, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) break;
            put(kst + s * kTile, kw, pg);
            if (warp == 8) {
                if (ct < 8) sm.sc[j & 3][ct] = sc;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.sc_full[j & 3]);
            }
            if (lane == 0) mbar_arrive(&sm.k_full[s]);
            if (warp == 8) sc = scales(j + 1);
            load(a.k, j + 1, pn, kw);
            if (j >= 2) ok = pr_wait(&sm.v_empty[s], ((j >> 1) - 1) & 1, a.status, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) break;
            put(vst + s * kTile, vw, pg);
            if (lane == 0) mbar_arrive(&sm.v_full[s]);
            #pragma unroll
            for (int i = 0; i < NP; ++i) pg[i] = pn[i];
        }
    } else if (lane == 0 && steps > 0) {
        // --- the products; a stage is handed back only where it will be filled again, so the last
        // arrival that is on its way is one that somebody waits for ---
        constexpr uint32_t idesc_s = umma_idesc_f16_f32(128, kPrKeys);
        constexpr uint32_t idesc_o = umma_idesc_f16_f32(128, D) | (1u << 16);  // V: MN-major
        const uint32_t q0 = smem_u32(qs), k0 = smem_u32(kst), v0 = smem_u32(vst);
        auto scores = [&](int t, int s) {
            #pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t at = uint32_t((i >> 2) * kBlk + (i & 3) * 32);
                umma_f16(tm + 128 * t, umma_desc_k_sw128(q0 + t * kTile + at), umma_desc_k_sw128(k0 + s * kTile + at),
                         idesc_s, i > 0);
            }
            umma_commit(&sm.s_full[t]);
        };
        bool ok = pr_wait(&sm.q_full, 0, a.status, abort_flag) && pr_wait(&sm.k_full[0], 0, a.status, abort_flag);
        tc_fence_after();
        if (ok) {
            for (int t = 0; t < nt; ++t) scores(t, 0);
            if (steps > 2) umma_commit(&sm.k_empty[0]);
        }
        for (int j = 0; ok && j < steps; ++j) {
            const int s = j & 1, sn = (j + 1) & 1;
            const bool more = j + 1 < steps;
            if (more) ok = pr_wait(&sm.k_full[sn], ((j + 1) >> 1) & 1, a.status, abort_flag);
            ok = ok && pr_wait(&sm.v_full[s], (j >> 1) & 1, a.status, abort_flag);
            for (int t = 0; ok && t < nt; ++t) {
                ok = pr_wait(&sm.p_full[t], j & 1, a.status, abort_flag);
                if (!ok) break;
                tc_fence_after();
                #pragma unroll
                for (int i = 0; i < kPrKeys / 16; ++i)
                    umma_f16_ts(tm + 256 + 128 * t, tm + 128 * t + 8 * i,
                                umma_desc_mn_sw128(v0 + s * kTile + 2048 * i, kBlk), idesc_o, j > 0 || i > 0);
                umma_commit(&sm.o_full[t]);
                if (more) scores(t, sn);
            }
            if (!ok) break;
            if (j + 2 < steps) umma_commit(&sm.v_empty[s]);
            if (j + 3 < steps) umma_commit(&sm.k_empty[sn]);
        }
        // after a wait that ran out: the products in flight still use TMEM and shared memory
        if (!ok) {
            mbar_init(&sm.q_full, 1);
            mbar_fence_init();
            umma_commit(&sm.q_full);
            mbar_wait(&sm.q_full, 0, a.status);
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tm, kPrTmem);
    }
    if (ns == 1) return;

    // --- join the parts of the keys: the CTA that ends last, in key order ---
    if (tid == 0) {
        int prev;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(a.counters + item) : "memory");
        sm.last = prev == ns - 1;
        if (prev == ns - 1) a.counters[item] = 0;  // ready for the next call
    }
    __syncthreads();
    if (!sm.last) return;
    const float* parts = a.part + item * args.splits * int64_t(kPrRows) * (D + 2);
    const int64_t pitch = int64_t(kPrRows) * (D + 2);
    float* wt = reinterpret_cast<float*>(qs);  // [ns][rows]
    for (int f = tid; f < rows; f += kPrThreads) {
        float mx = -INFINITY, sum = 0.f;
        for (int p = 0; p < ns; ++p) mx = fmaxf(mx, __ldcg(parts + p * pitch + f));
        for (int p = 0; p < ns; ++p) {
            const float w = mx == -INFINITY ? 0.f : ex2(__ldcg(parts + p * pitch + f) - mx);
            wt[p * kPrRows + f] = w;
            sum = fmaf(__ldcg(parts + p * pitch + kPrRows + f), w, sum);
        }
        sm.wt[f] = sum;
        const int64_t row = row0 + (col0 + f) / G;
        if (a.lse && row < a.q_rows)
            a.lse[row * a.heads + hk * G + (col0 + f) % G] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += kPrThreads) {
        const int f = i / (D / 4), d = 4 * (i % (D / 4));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll 4
        for (int p = 0; p < ns; ++p) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(parts + p * pitch + 2 * kPrRows + f * D + d));
            const float w = wt[p * kPrRows + f];
            v.x = fmaf(o.x, w, v.x), v.y = fmaf(o.y, w, v.y), v.z = fmaf(o.z, w, v.z), v.w = fmaf(o.w, w, v.w);
        }
        const float sum = sm.wt[f], inv = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t row = row0 + (col0 + f) / G;
        if (row >= a.q_rows) continue;
        uint2 w;
        if constexpr (BF16) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v.x * inv, v.y * inv), y = __floats2bfloat162_rn(v.z * inv, v.w * inv);
            w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
        } else {
            w = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
        }
        if (sum == 0.f) w = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(a.out + (row * a.heads + hk * G + (col0 + f) % G) * D + d) = w;
    }
}

// The host knows the rows in all, not the requests' own: at most one part
// tile more per request.  Fewer CTAs than SMs: the keys of a tile are split.
KvPromptPlan kv_prompt_plan(const KvAttendCall& c, int sms) {
    const int64_t group = c.heads / c.kv_heads;
    KvPromptPlan p;
    p.tiles = c.q_rows * group / kPrRows + c.requests;
    const int64_t items = p.tiles * c.kv_heads;
    p.splits = items > 0 && items * 2 <= sms ? int(sms / items) : 1;
    p.bytes = p.splits > 1 ? size_t(items) * p.splits * kPrRows * (c.dim + 2) * 4 : 0;
    return p;
}

template <bool E4M3, bool BF16, int D>
static cudaError_t launch_prompt(const PrArgs& a, unsigned grid, cudaStream_t s) {
    constexpr size_t smem = pr_smem_bytes<D>();
    static_assert(smem <= 227 * 1024, "shared memory");
    auto* kernel = kv_prompt_kernel<E4M3, BF16, D>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    kernel<<<grid, kPrThreads, smem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t run_kv_prompt(const KvAttendCall& c, const KvAttendArgs& args, const KvPromptPlan& p, cudaStream_t s) {
    PrArgs a;
    a.a = args, a.splits = p.splits;
    const int64_t n = p.tiles * c.kv_heads * p.splits;
    if (n <= 0) return cudaSuccess;
    if (n > INT32_MAX) return cudaErrorInvalidConfiguration;
    const unsigned grid = unsigned(n);
    const auto by_dim = [&](auto e4, auto bf) {
        constexpr bool E = decltype(e4)::value, B = decltype(bf)::value;
        return c.dim == 128 ? launch_prompt<E, B, 128>(a, grid, s) : launch_prompt<E, B, 64>(a, grid, s);
    };
    const bool bf16 = c.x_dtype == DT_BF16;
    if (c.e4m3) return bf16 ? by_dim(std::true_type(), std::true_type()) : by_dim(std::true_type(), std::false_type());
    return bf16 ? by_dim(std::false_type(), std::true_type()) : by_dim(std::false_type(), std::false_type());
}

}  // namespace exl3
