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
// weights are computed.  16 warps:
//   0-3, 4-7  one row per thread: running maximum, weights, sums (tiles 0 and 1)
//   8-11      codes of 128 keys from global memory to f16 in shared memory
//             (128-byte swizzle; K is a K-major operand, V an MN-major one: the same bytes)
//   12        an elected lane issues S = Q K^T and O += P V (tcgen05, fp32 in TMEM)
//   13-15     leave at once: they make up the warpgroup whose registers the first eight warps take
//             (184 a thread: a row's 128 scores are read from TMEM once and stay in registers)
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

constexpr int kPrThreads = 16 * 32;
constexpr int kPrKeys = 128;        // keys per step
constexpr int kPrRows = 256;        // query rows per CTA
constexpr int kPrScaleSlots = 4;
constexpr int kPrMaxSplits = 64;    // weights of the parts fit shared memory
constexpr float kPrSlack = 8.f;     // log2: growth of the maximum that is let pass
constexpr uint32_t kPrTmem = 512;

struct PrSmem {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], sc_full[kPrScaleSlots];
    uint32_t tmem;
    int abort_flag, last;
    int64_t scan[kPrThreads / 32];
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

// D[tmem] (+)= A B by one elected lane of a converged warp; A in shared memory or in TMEM
__device__ __forceinline__ void elect_umma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void elect_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void elect_commit(uint64_t* bar) {
    asm volatile(
        "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
        : "memory");
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

// 8 bytes, or zeros.  Volatile: the load stays where it is written, ahead of the waits it is to overlap.
__device__ __forceinline__ uint2 load_early(const uint8_t* p, bool get) {
    uint2 v;
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %3, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n"
        " @p ld.global.nc.v2.u32 {%0, %1}, [%2];\n}\n"
        : "=r"(v.x), "=r"(v.y) : "l"(p), "r"(int(get)));
    return v;
}

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

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // warp: uniform
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
    const uint32_t tm = __shfl_sync(0xffffffffu, sm.tmem, 0);
    // columns: S0 0, S1 128, O0 256, O1 384.  Registers: 512 x 128 at launch = 256 x 184 + 128 x 96 + 128 x 48
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;\n");
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
            // of scores: above 0 whatever the scales, so that -inf stays -inf
            auto factor = [&](float kscale) { return fmaxf(cfac * kscale, 1e-37f); };
            // Scores of 128 keys to weights.  `edge`: some row of the warp does not see all of them.
            auto weigh = [&](bool edge, int base, int j, const float4* sc) {
                uint32_t v[4][32];
                #pragma unroll
                for (int h = 0; h < 4; ++h) tmem_load32(ts + 32 * h, v[h]);
                #pragma unroll
                for (int h = 0; h < 4; ++h) tmem_load_wait(v[h]);
                if (edge) {
                    #pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        // bit i: key base + 16 g + i is seen
                        const int from = min(max(lo - base - 16 * g, 0), 16), to = min(max(hi - base - 16 * g, 0), 16);
                        uint32_t bits = ((1u << to) - 1u) & ~((1u << from) - 1u);
                        if (sc[g].w == 0.f) bits = 0u;
                        #pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (!(bits >> i & 1u)) v[g >> 1][16 * (g & 1) + i] = 0xff800000u;  // -inf
                    }
                }
                // the row's largest
                float mx = -INFINITY;
                #pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float4 s4 = sc[g];
                    float x[16];
                    #pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(v[g >> 1][16 * (g & 1) + i]);
                    #pragma unroll
                    for (int n = 8; n; n >>= 1)
                        #pragma unroll
                        for (int i = 0; i < n; ++i) x[i] = fmaxf(x[i], x[i + n]);
                    mx = fmaxf(mx, fmaf(x[0], factor(s4.x), s4.y));
                }
                if (__any_sync(0xffffffffu, mx > ref + kPrSlack || (ref == -INFINITY && mx > ref))) {
                    const float nref = fmaxf(ref, mx);
                    const float alpha = ref == nref ? 1.f : ex2(ref - nref);  // 0 where nothing has been seen
                    l *= alpha;
                    ref = nref;
                    if (j > 0) {
                        if (!__all_sync(0xffffffffu, pr_wait(&sm.o_full[t], (j - 1) & 1, a.status, abort_flag))) return false;
                        tc_fence_after();
                        #pragma unroll 1
                        for (int h = 0; h < D / 32; ++h) {
                            uint32_t o[32];
                            tmem_load32(to + 32 * h, o);
                            tmem_load_wait(o);
                            #pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_store32(to + 32 * h, o);
                        }
                    }
                }
                const float off = ref == -INFINITY ? 0.f : ref;
                #pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t p[16];
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 s4 = sc[2 * h + g];
                        const float f = factor(s4.x);
                        const float2 mul = make_float2(f, f), add = make_float2(s4.y - off, s4.y - off);
                        float2 sum = make_float2(0.f, 0.f);
                        #pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const float2 raw = make_float2(__uint_as_float(v[h][16 * g + i]), __uint_as_float(v[h][16 * g + i + 1]));
                            float2 x = fma2(raw, mul, add);
                            x = make_float2(ex2(x.x), ex2(x.y));
                            sum = add2(sum, x);
                            p[8 * g + i / 2] = pack_half2(x.x, x.y);
                        }
                        l = fmaf(sum.x + sum.y, s4.z, l);
                    }
                    tmem_store16(ts + 16 * h, p);
                }
                return true;
            };
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

                ok = weigh(edge, base, j, sc);
                if (!ok) break;
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
        named_bar_arrive(1, 288);
        if (ns == 1) return;

        // --- join the parts of the keys: the CTA that ends last, in key order ---
        named_bar_sync(2, 256);
        if (tid == 0) {
            int prev;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(a.counters + item) : "memory");
            sm.last = prev == ns - 1;
            if (prev == ns - 1) a.counters[item] = 0;  // ready for the next call
        }
        named_bar_sync(2, 256);
        if (!sm.last) return;
        const float* parts = a.part + item * args.splits * int64_t(kPrRows) * (D + 2);
        const int64_t pitch = int64_t(kPrRows) * (D + 2);
        float* wt = reinterpret_cast<float*>(smem);  // [ns][rows]
        for (int f = tid; f < rows; f += 256) {
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
        named_bar_sync(2, 256);
        for (int i = tid; i < rows * (D / 4); i += 256) {
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
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n");
        // --- codes to f16 ---
        // a thread takes 8 dims of each 64-dim block of a key: 8 lanes' 16-byte stores of one block
        // fall on 8 different places of a swizzled 128-byte row
        constexpr int NB = D / 64;
        constexpr int NP = 4;                // passes of 16 keys (of one page) to half a step
        const int ct = tid - 256, kr = ct >> 3, ch = ct & 7;
        const int32_t* row_table = a.table + int64_t(b) * a.width;
        // Of the 16 keys (lane & 7) of a step: whether the tile sees any, and their page as the
        // table has it.  It is looked at one step later, when its load has long arrived.
        auto key_of = [&](int j) { return key0 + j * kPrKeys + 16 * (lane & 7); };
        auto some = [&](int j) { return j < steps && key_of(j) + 16 > lo_all && key_of(j) < hi_all; };
        auto raw_page = [&](int j) { return some(j) ? __ldg(row_table + (key_of(j) >> a.shift)) : -1; };
        auto page_of = [&](int j, int raw) {
            const bool in = raw >= 0 && raw < a.pages;
            if (some(j) && !in) set_status(a.status, DEV_BAD_INDEX);
            return in ? raw : -1;
        };
        const int64_t page_bytes = (int64_t(Hk) * D) << a.shift;
        const int64_t mine = (int64_t(hk) * D << a.shift) + kr * D + ch * 8;
        auto load = [&](const uint8_t* codes, int j, int half, int pg, uint2 (&w)[NP][NB]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int key = key0 + j * kPrKeys + (half * NP + i) * 16, pi = __shfl_sync(0xffffffffu, pg, half * NP + i);
                const uint8_t* p = codes + pi * page_bytes + mine + (key & (P - 1)) * D;
                // keys that no row sees are zeros: their codes may be NaN, and 0 * NaN is not 0
                const bool get = pi >= 0 && key + kr >= lo_all && key + kr < hi_all;
                #pragma unroll
                for (int n = 0; n < NB; ++n) w[i][n] = load_early(p + 64 * n, get);
            }
        };
        const uint32_t place = uint32_t(kr * 128 + ((ch ^ (kr & 7)) << 4));
        auto put = [&](char* dst, int half, const uint2 (&w)[NP][NB]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i)
                #pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t x = code_word<E4M3>(w[i][n].x), y = code_word<E4M3>(w[i][n].y);
                    *reinterpret_cast<uint4*>(dst + n * kBlk + (half * NP + i) * (16 * 128) + place) =
                        make_uint4(half2_lo<E4M3>(x), half2_hi<E4M3>(x), half2_lo<E4M3>(y), half2_hi<E4M3>(y));
                }
        };
        auto handed = [&](uint64_t* bar) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        float ks = 0.f, vs = 1.f;  // of lanes 0-7 of warp 8: their 16 keys' scales
        auto scales = [&](int pg) {
            if (warp != 8 || pg < 0) return;
            ks = __ldg(a.k_scale + int64_t(pg) * Hk + hk);
            vs = __ldg(a.v_scale + int64_t(pg) * Hk + hk);
        };
        // two halves are on their way while a third is written
        uint2 k0[NP][NB], k1[NP][NB], v0[NP][NB], v1[NP][NB];
        int pg = page_of(0, raw_page(0)), raw = raw_page(1);
        load(a.k, 0, 0, pg, k0);
        load(a.k, 0, 1, pg, k1);
        scales(pg);
        for (int j = 0; j < steps; ++j) {
            const int s = j & 1;
            bool ok = j < 2 || pr_wait(&sm.k_empty[s], ((j >> 1) - 1) & 1, a.status, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) break;
            put(kst + s * kTile, 0, k0);
            load(a.v, j, 0, pg, v0);
            put(kst + s * kTile, 1, k1);
            load(a.v, j, 1, pg, v1);
            if (warp == 8) {
                const int ve = stored_exponent(vs);
                if (lane < 8)
                    sm.sc[j & 3][lane] = pg < 0 ? make_float4(0.f, 0.f, 1.f, some(j) ? 0.f : 1.f)
                                                : make_float4(ks, float(ve), exp2_int(-ve), 1.f);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.sc_full[j & 3]);
            }
            handed(&sm.k_full[s]);
            pg = page_of(j + 1, raw);
            raw = raw_page(j + 2);
            scales(pg);
            ok = j < 2 || pr_wait(&sm.v_empty[s], ((j >> 1) - 1) & 1, a.status, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) break;
            put(vst + s * kTile, 0, v0);
            load(a.k, j + 1, 0, pg, k0);
            put(vst + s * kTile, 1, v1);
            load(a.k, j + 1, 1, pg, k1);
            handed(&sm.v_full[s]);
        }
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");
      if (warp > 12) return;
      if (steps > 0) {
        // --- the products.  The whole warp runs this, so that addresses stay in uniform registers; an
        // elected lane issues.  A stage is handed back only where it will be filled again, so the last
        // arrival on its way is one that somebody waits for ---
        constexpr uint32_t idesc_s = umma_idesc_f16_f32(128, kPrKeys);
        constexpr uint32_t idesc_o = umma_idesc_f16_f32(128, D) | (1u << 16);  // V: MN-major
        constexpr uint32_t kStep = kTile >> 4;
        const uint64_t q0 = umma_desc_k_sw128(smem_u32(qs)), k0 = umma_desc_k_sw128(smem_u32(kst));
        const uint64_t v0 = umma_desc_mn_sw128(smem_u32(vst), kBlk);
        auto scores = [&](int t, int s) {
            const uint64_t qd = q0 + uint32_t(t) * kStep, kd = k0 + uint32_t(s) * kStep;
            #pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t at = uint32_t((i >> 2) * kBlk + (i & 3) * 32) >> 4;
                elect_umma_ss(tm + 128 * t, qd + at, kd + at, idesc_s, i > 0);
            }
            elect_commit(&sm.s_full[t]);
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            return __all_sync(0xffffffffu, pr_wait(bar, parity, a.status, abort_flag)) != 0;
        };
        bool ok = wait(&sm.q_full, 0) && wait(&sm.k_full[0], 0);
        tc_fence_after();
        if (ok) {
            for (int t = 0; t < nt; ++t) scores(t, 0);
            if (steps > 2) elect_commit(&sm.k_empty[0]);
        }
        for (int j = 0; ok && j < steps; ++j) {
            const int s = j & 1, sn = (j + 1) & 1;
            const bool more = j + 1 < steps;
            if (more) ok = wait(&sm.k_full[sn], ((j + 1) >> 1) & 1);
            ok = ok && wait(&sm.v_full[s], (j >> 1) & 1);
            for (int t = 0; ok && t < nt; ++t) {
                ok = wait(&sm.p_full[t], j & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = v0 + uint32_t(s) * kStep;
                #pragma unroll
                for (int i = 0; i < kPrKeys / 16; ++i)
                    elect_umma_ts(tm + 256 + 128 * t, tm + 128 * t + 8 * i, vd + uint32_t(2048 * i >> 4), idesc_o,
                                  i > 0 ? 1u : uint32_t(j > 0));
                elect_commit(&sm.o_full[t]);
                if (more) scores(t, sn);
            }
            if (!ok) break;
            if (j + 2 < steps) elect_commit(&sm.v_empty[s]);
            if (j + 3 < steps) elect_commit(&sm.k_empty[sn]);
        }
        // after a wait that ran out: the products in flight still use TMEM and shared memory
        if (!ok) {
            if (lane == 0) {
                mbar_init(&sm.q_full, 1);
                mbar_fence_init();
            }
            __syncwarp();
            elect_commit(&sm.q_full);
            mbar_wait(&sm.q_full, 0, a.status);
        }
      }
      __syncwarp();
      named_bar_sync(1, 288);  // the rows are read
      tc_fence_after();
      tmem_dealloc(tm, kPrTmem);
    }
}

// The host knows the rows in all, not the requests' own: at most one part
// tile more per request.  Fewer CTAs than SMs: the keys of a tile are split.
KvPromptPlan kv_prompt_plan(const KvAttendCall& c, int sms) {
    const int64_t group = c.heads / c.kv_heads;
    KvPromptPlan p;
    p.tiles = c.q_rows * group / kPrRows + c.requests;
    const int64_t items = p.tiles * c.kv_heads;
    p.splits = items > 0 && items * 2 <= sms ? int(sms / items < kPrMaxSplits ? sms / items : kPrMaxSplits) : 1;
    p.bytes = p.splits > 1 ? size_t(items) * p.splits * kPrRows * (c.dim + 2) * 4 : 0;
    return p;
}

template <bool E4M3, bool BF16, int D>
static cudaError_t launch_prompt(const PrArgs& a, unsigned grid, cudaStream_t s) {
    constexpr size_t smem = pr_smem_bytes<D>();
    static_assert(smem <= 227 * 1024 && kPrMaxSplits * kPrRows * 4 + sizeof(PrSmem) + 1024 <= smem, "shared memory");
    auto* kernel = kv_prompt_kernel<E4M3, BF16, D>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = raise_smem(kernel, smem, done);
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
