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
//   13        pages and scales of the steps to come, four steps at a time, into a ring
//   14        the items to come into another: what every warp needs to know of them stays in shared memory
//   12        an elected lane issues S = Q K^T and O += P V (tcgen05, fp32 in TMEM)
//   15        idle: it makes up the warpgroup whose registers the first eight warps take
//             (184 a thread: a row's 128 scores are read from TMEM once and stay in registers)
// TMEM: S0 S1 (128 columns each; the weights, f16, take the place of the
// scores that they came from and are the A operand of P V), O0 O1.
// The order of the issue S0 S1 | PV0 S0' PV1 S1' | ... keeps one tile's
// products behind the other's weights; tcgen05 runs one thread's products in order.
//
// Work: an item is (request, 256 rows, kv head), its steps are the 128-key
// blocks that its rows see; all items' steps, and a few for each item's start
// and end, form one line that the CTAs, one per SM, split evenly, whatever the
// lengths and the causal mask.  (Steps alone give a prompt's first rows, whose
// items have one or two, to too few CTAs.)  An item cut
// by a CTA boundary is joined from fp32 partials by the CTA that finishes it
// last, in key order.  (A least number of steps per CTA does not pay: a prompt
// of 256 rows of 8 heads took 49 us with four, 30 with two, 27 with one.)
//
// Measured (lone calls): a prompt's last 4096 tokens of 16384 (32 heads over 4,
// dim 128, e4m3) 1.03 ms, 935 TFLOP/s (56 % of the measured bf16 rate); in a graph,
// inputs partly in L2, 0.99.  No single unit bounds it: without its
// exponentials it takes 1036 of then 1064 us, with an eighth of the products 1003,
// without loads 1077.  It is the chain of a tile's scores, weights, product
// and next scores, with three warps per scheduler at 0.4 instructions a clock.
// Five prompts of up to 1777 tokens, window 1000 (24 heads over 8, dim 64, int8)
// 145 us, 138 in a graph: 4.7 items of 9 steps a CTA, and at each item's start
// and end (queries in, first scores, last output out) the units wait; a third of the
// CTAs' steps and a quarter of the warps' have masks.
// Registers decide much: a converter or an issuing warp that spills costs up to 40 %.
//
// O is rescaled only when a row's maximum grows by more than 2^8 over the
// place that its weights' reference was set for (kAttLift, kAttSlack): until then
// larger weights (f16 holds them, the sums are fp32) cost nothing, and the
// final division is by a sum over the same reference.
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
constexpr int kPrSlots = 8;         // steps whose pages and scales are kept
constexpr uint32_t kPrTmem = 512;
// Steps that an item's queries and results are worth on the line.  us with 0 / 3 / 6 / 10:
//   whole prompts of 2043 to 4086 tokens (16 heads over 4, dim 128, int8) 478 / 280 / 286 / 300, one of 4086 228 / 117 / 122 / 129
//   six of 1337 to 2673 tokens (24 heads over 8, e4m3), dim 128 603 / 382 / 398 / 418, dim 64 421 / 311 / 326 / 338
//   up to 2000 tokens behind a prefix, 8000 in all 297 / 280 / 276 / 284
constexpr int kPrItemCost = 3;

// pages and scales of a step
struct PrStep {
    float4 sc[8];  // of 16 keys: K scale, log2 V scale, 1 / V scale, 1 if the page exists
    int64_t at[8];  // of 16 keys: where their codes begin, -1: not seen, or no such page
    int from, count;  // the keys of the step that any row sees
};

// an item's share of this CTA: `steps` of its `all` steps, from `off` on
struct PrItem {
    int64_t row0, col0;
    int steps, off, all;  // steps 0: no more items
    int rows, hk, first, keys, k_begin;
    int c0, c1;           // the CTAs that share the item
};
constexpr int kPrItems = 4;

struct PrSmem {
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    uint64_t step_full[kPrSlots], step_free[kPrSlots], item_full[kPrItems], item_free[kPrItems];
    uint64_t join[2];  // of a tile's rows among themselves
    uint64_t done;
    uint32_t tmem;
    int abort_flag, last[2];
    int64_t scan[kPrThreads / 32];
    int found_b, found_tile, tile_index;  // of the CTA's first step: request, its tile, the tile's place among all
    int64_t found_base;                   // that tile's first step
    int64_t steps_from, steps_upto;       // the CTA's steps
    int64_t line;                         // length of the line
    PrStep step[kPrSlots];
    PrItem item[kPrItems];
};

template <int D>
constexpr size_t pr_smem_bytes() {
    return 1024 + size_t(kPrRows) * D * 2 + 4 * size_t(kPrKeys) * D * 2 + sizeof(PrSmem);
}
static_assert((4 * kPrKeys + kPrRows) * 64 * 2 >= (kKvMaxRequests + 1) * 4, "the tile sums fit the place of the operands");

// fp32 partial of one 128-row tile: {reference, sum} per row, then O in 16-byte pieces, rows side by side
template <int D>
__host__ __device__ constexpr int pr_part() { return 128 * (D + 2); }

// Waits for a phase.  One that runs out of its budget records the status and
// raises the flag, after which no wait waits: every loop here ends by itself, so
// the kernel runs through (its results are void) and no warp is left behind.
__device__ __forceinline__ void pr_wait(uint64_t* bar, uint32_t parity, int* status, volatile int* abort_flag) {
    const uint32_t addr = smem_u32(bar);
    auto ready = [&]() {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
        return ok != 0;
    };
    if (ready()) return;
    const long long t0 = clock64();
    while (!ready()) {
        if (*abort_flag) return;
        if (clock64() - t0 > kWaitBudgetCycles) {
            set_status(status, DEV_WAIT_TIMEOUT);
            *abort_flag = 1;
            return;
        }
    }
}

__device__ __forceinline__ int pr_tiles(const KvAttendArgs& a, int b) {
    const int64_t cols = int64_t(att_rows(a, b).rows) * a.group;
    return cols > a.few ? int((cols + kPrRows - 1) / kPrRows) : 0;
}

// 256 rows of a request and the keys that any of them sees
struct PrTile {
    int64_t row0, col0;
    int first, keys, rows, lo, hi, k_begin, steps;  // first: position of the request's first row
};
__device__ __forceinline__ PrTile pr_tile(const KvAttendArgs& a, int b, int tile) {
    PrTile t;
    const AttRows w = att_rows(a, b);
    t.row0 = w.row0;
    const int len = max(a.kv_lens[b], 0);
    t.keys = att_keys(a, len), t.first = len - w.fresh;
    t.col0 = int64_t(tile) * kPrRows;
    t.rows = int(min(int64_t(w.rows) * a.group - t.col0, int64_t(kPrRows)));
    const int first = t.first + int(t.col0 / a.group), last = t.first + int((t.col0 + t.rows - 1) / a.group);
    t.hi = max(min(last + 1, t.keys), 0);
    t.lo = min(a.window > 0 ? max(first + 1 - a.window, 0) : 0, t.hi);
    t.k_begin = t.lo & ~15;  // pages and scales are looked up by 16 keys
    t.steps = max((t.hi - t.k_begin + kPrKeys - 1) / kPrKeys, 1);  // rows that see nothing take one step too
    return t;
}

// A place on the line of steps, ordered by request, tile, kv head, keys
struct PrWalk {
    int64_t base;  // of the tile's first step
    int b, tile, tiles, index;
    PrTile t;
    __device__ __forceinline__ void start(const KvAttendArgs& a, const PrSmem& sm) {
        base = sm.found_base, b = sm.found_b, tile = sm.found_tile, index = sm.tile_index;
        tiles = pr_tiles(a, b);
        t = pr_tile(a, b, tile);
    }
    __device__ __forceinline__ void seek(const KvAttendArgs& a, int64_t u) {  // forwards, to a step below the total
        while (u >= base + int64_t(a.kv_heads) * t.steps) {
            base += int64_t(a.kv_heads) * t.steps;
            ++index;
            if (++tile >= tiles) {
                do tiles = pr_tiles(a, ++b);
                while (tiles == 0);
                tile = 0;
            }
            t = pr_tile(a, b, tile);
        }
    }
};

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

// D[tmem] (+)= A B by one elected lane of a converged warp; A in shared memory or in TMEM.  Descriptors
// come as their low words (address, leading offset); `hi` is the high word that all of a kind share.
__device__ __forceinline__ void elect_umma_ss(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 da, db;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
        " elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}\n" ::"r"(tmem_d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void elect_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 db;\n mov.b64 db, {%2, %3};\n"
        " elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %5, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(tmem_d),
        "r"(tmem_a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
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

// the largest of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <bool INC, int N>
__device__ __forceinline__ void set_registers() {
    if constexpr (INC) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(kPrThreads, 1) kv_prompt_kernel(const KvAttendArgs a) {
    constexpr int kBlk = kPrKeys * 128;        // bytes of a 64-dim block of 128 rows
    constexpr int kTile = (D / 64) * kBlk;     // a 128-row f16 tile
    // Registers a thread: 512 x 128 at launch are handed out as 256 rows', 128 codes', 128 others'
    constexpr int kRowRegs = D == 128 ? 184 : 192, kCodeRegs = D == 128 ? 96 : 80, kRestRegs = 48;
    static_assert(2 * kRowRegs + kCodeRegs + kRestRegs == 512, "what the launch has");
    extern __shared__ char pr_raw[];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(pr_raw) + 1023) & ~uintptr_t(1023));
    char* vst = smem;              // 2 stages
    char* kst = vst + 2 * kTile;   // 2 stages
    char* qs = kst + 2 * kTile;    // 2 tiles
    PrSmem& sm = *reinterpret_cast<PrSmem*>(qs + 2 * kTile);
    volatile int* abort_flag = &sm.abort_flag;

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // warp: uniform
    const int Hk = a.kv_heads, G = a.group, P = 1 << a.shift;

    // --- this CTA's share of the line of steps ---
    // Block-wide sum of one value per thread; returns the sum of the threads up to and with this one
    auto scan = [&](int64_t v, int64_t& total) {
        #pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += o;
        }
        if (lane == 31) sm.scan[warp] = v;
        __syncthreads();
        total = 0;
        for (int w = 0; w < kPrThreads / 32; ++w) {
            if (w == warp) v += total;
            total += sm.scan[w];
        }
        __syncthreads();
        return v;
    };
    int32_t* sums = reinterpret_cast<int32_t*>(smem);  // [requests + 1] tiles of the requests before; the operands come later
    int ctas;
    {
        const int per = (a.requests + kPrThreads - 1) / kPrThreads;
        int64_t mine = 0, n_tiles, total;
        for (int i = 0; i < per; ++i)
            if (tid * per + i < a.requests) mine += pr_tiles(a, tid * per + i);
        int64_t at = scan(mine, n_tiles) - mine;
        for (int i = 0; i < per; ++i)
            if (tid * per + i < a.requests) {
                sums[tid * per + i] = int32_t(at);
                at += pr_tiles(a, tid * per + i);
            }
        if (tid == 0) sums[a.requests] = int32_t(n_tiles);
        __syncthreads();
        const int each = int((n_tiles + kPrThreads - 1) / kPrThreads);
        const int64_t t0 = int64_t(tid) * each, t1 = min(t0 + each, n_tiles);
        auto request = [&](int64_t t) {  // of tile t: the last b with sums[b] <= t
            int lo = 0, hi = a.requests;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sums[mid] <= t) lo = mid;
                else hi = mid;
            }
            return lo;
        };
        mine = 0;
        for (int64_t t = t0; t < t1; ++t) {
            const int b = request(t);
            mine += int64_t(Hk) * pr_tile(a, b, int(t - sums[b])).steps;
        }
        const int64_t end = scan(mine, total);
        // Step s of item i (all counted from 0) is at s + (i + 1) kPrItemCost of the line
        const int64_t line = total + int64_t(kPrItemCost) * Hk * n_tiles;
        ctas = int(min(int64_t(gridDim.x), total));
        if (int(blockIdx.x) >= ctas) return;
        if (tid == 0) sm.line = line, sm.steps_upto = total;
        __syncthreads();
        const int64_t u0 = line * blockIdx.x / ctas, u1 = line * (blockIdx.x + 1) / ctas;
        auto at_line = [&](int64_t step, int64_t t) { return step + int64_t(kPrItemCost) * Hk * t; };
        const int64_t from = at_line(end - mine, min(t0, n_tiles)), upto = at_line(end, max(t1, t0));
        const bool has0 = t0 < t1 && u0 >= from && u0 < upto, has1 = t0 < t1 && u1 >= from && u1 < upto;
        if (has0 || has1) {
            int64_t base = end - mine;
            for (int64_t t = t0; t < t1; ++t) {
                const int b = request(t);
                const int64_t tile_steps = pr_tile(a, b, int(t - sums[b])).steps;
                // steps before place u of the line
                auto steps_before = [&](int64_t u) {
                    const int64_t o = u - at_line(base, t), item = tile_steps + kPrItemCost, head = o / item;
                    return base + head * tile_steps + max(o - head * item - kPrItemCost, int64_t(0));
                };
                auto inside = [&](int64_t u) { return u >= at_line(base, t) && u < at_line(base + Hk * tile_steps, t + 1); };
                if (has0 && inside(u0)) {
                    sm.found_b = b, sm.found_tile = int(t - sums[b]), sm.found_base = base, sm.tile_index = int(t);
                    sm.steps_from = steps_before(u0);
                }
                if (has1 && inside(u1)) sm.steps_upto = steps_before(u1);
                base += Hk * tile_steps;
            }
        }
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.q_full[i], 128);
            mbar_init(&sm.k_full[i], 4);
            mbar_init(&sm.v_full[i], 4);
            mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.o_full[i], 1);
            mbar_init(&sm.p_full[i], 128);
            mbar_init(&sm.join[i], 128);
        }
        for (int i = 0; i < kPrSlots; ++i) {
            mbar_init(&sm.step_full[i], 1);
            mbar_init(&sm.step_free[i], 4);
        }
        for (int i = 0; i < kPrItems; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_free[i], 9);  // the rows' warps and the products'
        }
        mbar_init(&sm.done, 1);
        sm.abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    const int64_t u0 = sm.steps_from, u1 = sm.steps_upto, line = sm.line;  // this CTA's steps
    if (u0 >= u1) return;  // its part of the line has none
    if (warp == 12) tmem_alloc(&sm.tmem, kPrTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = __shfl_sync(0xffffffffu, sm.tmem, 0);
    const int cta = blockIdx.x;
    // TMEM columns: S0 0, S1 128, O0 256, O1 384
    if (warp < 8) {
        set_registers<true, kRowRegs>();
        const int t = warp >> 2, r = tid & 127, f = t * 128 + r;
        const uint32_t lane_base = uint32_t(32 * (warp & 3)) << 16;
        const uint32_t ts = tm + lane_base + uint32_t(128 * t), to = tm + lane_base + uint32_t(256 + 128 * t);
        uint32_t n = 0;    // steps of this CTA so far
        uint32_t nt_n = 0; // those that this tile took part in
        uint32_t joins = 0;
        for (uint32_t it = 0;; ++it) {
            const PrItem& im = sm.item[it % kPrItems];
            pr_wait(&sm.item_full[it % kPrItems], (it / kPrItems) & 1, a.status, abort_flag);
            if (__any_sync(0xffffffffu, *abort_flag)) break;
            const int steps = im.steps;
            if (steps == 0) break;
            auto leave = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.item_free[it % kPrItems]);
            };
            if (t * 128 >= im.rows) {  // the request's last tile is a narrow one
                n += steps;
                leave();
                continue;
            }
            // --- this thread's row ---
            const int64_t fc = im.col0 + f, row = im.row0 + fc / G;
            const bool mine = f < im.rows;
            const int64_t at = row * a.heads + im.hk * G + fc % G;
            float cfac = fabsf(a.scale_log2);
            {
                const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;  // group maxima below need a factor >= 0
                const uint4* qp = reinterpret_cast<const uint4*>(a.q + (mine ? row * a.q_tok + int64_t(im.hk * G + fc % G) * a.q_head : 0));
                uint4 x[D / 8];
                #pragma unroll
                for (int i = 0; i < D / 8; ++i) x[i] = mine ? __ldg(qp + i) : make_uint4(0, 0, 0, 0);
                float mul = sign;
                if constexpr (BF16) {
                    // to f16 by a power of two per row: largest magnitude in [2^14, 2^15), so that
                    // values down to 2^-31 of it keep all 8 bits
                    uint32_t m2 = 0;
                    #pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu),
                                                   __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu)));
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
                    // the products that read the tile's last rows here are done: this thread has waited for the outputs after them
                    *reinterpret_cast<uint4*>(qs + t * kTile + (i >> 3) * kBlk + r * 128 + (((i & 7) ^ (r & 7)) << 4)) =
                        make_uint4(conv(x[i].x), conv(x[i].y), conv(x[i].z), conv(x[i].w));
                }
                fence_async_smem();
                tc_fence_before();
                mbar_arrive(&sm.q_full[t]);
            }
            const int pos = im.first + int(fc / G);
            const int hi = mine ? min(pos + 1, im.keys) : 0;
            const int lo = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
            float ref = -INFINITY, l = 0.f;
            // of scores: above 0 whatever the scales, so that -inf stays -inf
            auto factor = [&](float kscale) { return fmaxf(cfac * kscale, 1e-37f); };
            int base = im.k_begin + im.off * kPrKeys;
            for (int j = 0; j < steps; ++j, ++n, ++nt_n, base += kPrKeys) {
                const PrStep& st = sm.step[n % kPrSlots];
                pr_wait(&sm.step_full[n % kPrSlots], (n / kPrSlots) & 1, a.status, abort_flag);
                pr_wait(&sm.s_full[t], nt_n & 1, a.status, abort_flag);
                __syncwarp();
                tc_fence_after();
                // the row's scores, read once
                uint32_t v[4][32];
                #pragma unroll
                for (int h = 0; h < 4; ++h) tmem_load32(ts + 32 * h, v[h]);
                bool dead = mine && (base + kPrKeys > hi || base < lo);  // rows past the tile's end see nothing and give nothing
                #pragma unroll
                for (int g = 0; g < 8; ++g) dead |= st.sc[g].w == 0.f;
                const bool edge = __any_sync(0xffffffffu, dead);  // some row of the warp does not see all of them
                auto mask = [&](int h, uint32_t (&x)[32]) {
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        // bit i: key base + 32 h + 16 g + i is seen
                        const int k0 = base + 32 * h + 16 * g;
                        const int from = min(max(lo - k0, 0), 16), upto = min(max(hi - k0, 0), 16);
                        uint32_t bits = ((1u << upto) - 1u) & ~((1u << from) - 1u);
                        if (st.sc[2 * h + g].w == 0.f) bits = 0u;
                        #pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (!(bits >> i & 1u)) x[16 * g + i] = 0xff800000u;  // -inf
                    }
                };
                float mx = -INFINITY;
                #pragma unroll
                for (int h = 0; h < 4; ++h) {
                    tmem_load_wait(v[h]);
                    if (edge) mask(h, v[h]);
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 s4 = st.sc[2 * h + g];
                        auto x = [&](int i) { return __uint_as_float(v[h][16 * g + i]); };
                        const float m0 = max3(x(0), x(1), x(2)), m1 = max3(x(3), x(4), x(5)), m2 = max3(x(6), x(7), x(8));
                        const float m3 = max3(x(9), x(10), x(11)), m4 = max3(x(12), x(13), x(14));
                        const float top = max3(max3(m0, m1, m2), max3(m3, m4, x(15)), -INFINITY);
                        mx = max3(mx, fmaf(top, factor(s4.x), s4.y), -INFINITY);
                    }
                }
                if (__any_sync(0xffffffffu, mx > ref + (kAttLift + kAttSlack))) {  // -inf + slack is -inf: the first key that is seen counts as growth
                    const float nref = fmaxf(ref, mx - kAttLift);  // of a NaN row: any
                    const float alpha = ref == nref ? 1.f : ex2(ref - nref);  // 0 where nothing has been seen
                    l *= alpha;
                    ref = nref;
                    if (j > 0) {
                        pr_wait(&sm.o_full[t], (nt_n - 1) & 1, a.status, abort_flag);
                        __syncwarp();
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
                const float less = ref == -INFINITY ? 0.f : ref;
                #pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t p[16];
                    #pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4 s4 = st.sc[2 * h + g];
                        const float fg = factor(s4.x);
                        const float2 mul = make_float2(fg, fg), add = make_float2(s4.y - less, s4.y - less);
                        float2 sum = make_float2(0.f, 0.f);
                        #pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const float2 raw = make_float2(__uint_as_float(v[h][16 * g + i]), __uint_as_float(v[h][16 * g + i + 1]));
                            const float2 x = fma2(raw, mul, add);
                            const float2 e = make_float2(ex2(x.x), ex2(x.y));
                            sum = add2(sum, e);
                            p[8 * g + i / 2] = pack_half2(e.x, e.y);
                        }
                        l = fmaf(sum.x + sum.y, s4.z, l);
                    }
                    tmem_store16(ts + 16 * h, p);
                }
                tmem_store_wait();
                tc_fence_before();
                mbar_arrive(&sm.p_full[t]);
            }
            // --- the row's result ---
            pr_wait(&sm.o_full[t], (nt_n - 1) & 1, a.status, abort_flag);
            __syncwarp();
            tc_fence_after();
            // 32 dims of a row from h on
            auto emit = [&](int h, const float (&o)[32], float inv) {
                uint32_t x[16];
                #pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (BF16) {
                        const __nv_bfloat162 q2 = __floats2bfloat162_rn(o[2 * i] * inv, o[2 * i + 1] * inv);
                        x[i] = *reinterpret_cast<const uint32_t*>(&q2);
                    } else {
                        x[i] = pack_half2(o[2 * i] * inv, o[2 * i + 1] * inv);
                    }
                    if (inv == 0.f) x[i] = 0u;
                }
                uint4* dst = reinterpret_cast<uint4*>(a.out + at * D + 32 * h);
                if (mine)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) dst[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            };
            auto emit_lse = [&](float m, float sum) {
                if (mine && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
            };
            const bool whole = steps == im.all;
            float* part = a.part + (int64_t(2 * cta + (im.off == 0 ? 1 : 0)) * 2 + t) * pr_part<D>();
            if (!whole) {
                __stcg(part + r, ref);
                __stcg(part + 128 + r, l);
            }
            #pragma unroll 1
            for (int h = 0; h < D / 32; ++h) {
                uint32_t o[32];
                tmem_load32(to + 32 * h, o);
                tmem_load_wait(o);
                float x[32];
                #pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(o[i]);
                if (whole) {
                    emit(h, x, l == 0.f ? 0.f : 1.f / l);  // a row that sees no key is zero
                } else {
                    float4* dst = reinterpret_cast<float4*>(part + 256) + 8 * h * 128 + r;
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) __stcg(dst + i * 128, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
                }
            }
            if (whole) {
                emit_lse(ref, l);
                leave();
                continue;
            }
            // --- join the parts: the CTA that ends last, in key order ---
            const int c0 = im.c0, c1 = im.c1;
            // the tile's 128 threads; bounded like every other wait, since a warp may have given up before
            auto together = [&]() {
                mbar_arrive(&sm.join[t]);
                pr_wait(&sm.join[t], joins++ & 1, a.status, abort_flag);
            };
            together();
            if (r == 0) {
                int prev;
                int32_t* counter = a.counters + 2 * c0 + t;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(counter) : "memory");
                sm.last[t] = prev == c1 - c0;
                if (prev == c1 - c0) *counter = 0;  // ready for the next call
            }
            together();
            if (sm.last[t]) {
                auto piece = [&](int c) { return a.part + (int64_t(2 * c + (c == c0 ? 1 : 0)) * 2 + t) * pr_part<D>(); };
                float m = -INFINITY, sum = 0.f;
                #pragma unroll 4
                for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(piece(c) + r));
                const float less = m == -INFINITY ? 0.f : m;
                #pragma unroll 4
                for (int c = c0; c <= c1; ++c) sum = fmaf(__ldcg(piece(c) + 128 + r), ex2(__ldcg(piece(c) + r) - less), sum);
                #pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    float x[32];
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = 0.f;
                    #pragma unroll 1
                    for (int c = c0; c <= c1; ++c) {
                        const float* pc = piece(c);
                        const float wc = ex2(__ldcg(pc + r) - less);
                        const float4* src = reinterpret_cast<const float4*>(pc + 256) + 8 * h * 128 + r;
                        #pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 o = __ldcg(src + i * 128);
                            x[4 * i] = fmaf(o.x, wc, x[4 * i]), x[4 * i + 1] = fmaf(o.y, wc, x[4 * i + 1]);
                            x[4 * i + 2] = fmaf(o.z, wc, x[4 * i + 2]), x[4 * i + 3] = fmaf(o.w, wc, x[4 * i + 3]);
                        }
                    }
                    emit(h, x, sum == 0.f ? 0.f : 1.f / sum);
                }
                emit_lse(m, sum);
            }
            together();  // sm.last is the next item's
            leave();
        }
        tc_fence_before();
        named_bar_arrive(1, 288);
    } else if (warp < 12) {
        set_registers<false, kCodeRegs>();
        // --- codes to f16 ---
        // a thread takes 8 dims of each 64-dim block of a key: 8 lanes' 16-byte stores of one block
        // fall on 8 different places of a swizzled 128-byte row
        constexpr int NB = D / 64;
        constexpr int NP = 4;                // passes of 16 keys (of one page) to half a step
        const int ct = tid - 256, kr = ct >> 3, ch = ct & 7;
        const uint8_t* const k_mine = a.k + kr * D + ch * 8;
        const uint8_t* const v_mine = a.v + kr * D + ch * 8;
        auto load = [&](const uint8_t* codes, const PrStep& st, int half, uint2 (&w)[NP][NB]) {
            const uint32_t first = uint32_t(half * NP * 16 + kr - st.from), count = uint32_t(st.count);
            #pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int64_t at = st.at[half * NP + i];
                // keys that no row sees are zeros: their codes may be NaN, and 0 * NaN is not 0
                const bool get = at >= 0 && first + 16 * i < count;
                #pragma unroll
                for (int m = 0; m < NB; ++m) w[i][m] = load_early(codes + at + 64 * m, get);
            }
        };
        const uint32_t place = uint32_t(kr * 128 + ((ch ^ (kr & 7)) << 4));
        auto put = [&](char* dst, int half, const uint2 (&w)[NP][NB]) {
            #pragma unroll
            for (int i = 0; i < NP; ++i)
                #pragma unroll
                for (int m = 0; m < NB; ++m) {
                    const uint32_t x = code_word<E4M3>(w[i][m].x), y = code_word<E4M3>(w[i][m].y);
                    *reinterpret_cast<uint4*>(dst + m * kBlk + (half * NP + i) * (16 * 128) + place) =
                        make_uint4(half2_lo<E4M3>(x), half2_hi<E4M3>(x), half2_lo<E4M3>(y), half2_hi<E4M3>(y));
                }
        };
        auto handed = [&](uint64_t* bar) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        const uint32_t steps = uint32_t(u1 - u0);
        auto known = [&](uint32_t n) {  // false after a wait that ran out: the slot may hold anything
            pr_wait(&sm.step_full[n % kPrSlots], (n / kPrSlots) & 1, a.status, abort_flag);
            return !__any_sync(0xffffffffu, *abort_flag);
        };
        // two halves are on their way while a third is written
        uint2 k0[NP][NB], k1[NP][NB], v0[NP][NB], v1[NP][NB];
        if (known(0)) {
            load(k_mine, sm.step[0], 0, k0);
            load(k_mine, sm.step[0], 1, k1);
            for (uint32_t n = 0; n < steps; ++n) {
                const uint32_t s = n & 1;
                if (n >= 2) pr_wait(&sm.k_empty[s], ((n >> 1) - 1) & 1, a.status, abort_flag);
                __syncwarp();
                const PrStep& st = sm.step[n % kPrSlots];
                put(kst + s * kTile, 0, k0);
                load(v_mine, st, 0, v0);
                put(kst + s * kTile, 1, k1);
                load(v_mine, st, 1, v1);
                handed(&sm.k_full[s]);
                // K of step n is in place of step n - 2's, whose products, and those of n - 3's weights, are
                // done: every row has left step n - 3, and its slot is free
                if (n >= 3 && lane == 0) mbar_arrive(&sm.step_free[(n - 3) % kPrSlots]);
                const bool more = n + 1 < steps;
                if (more && !known(n + 1)) break;
                if (n >= 2) pr_wait(&sm.v_empty[s], ((n >> 1) - 1) & 1, a.status, abort_flag);
                __syncwarp();
                const PrStep& next = sm.step[(n + 1) % kPrSlots];
                put(vst + s * kTile, 0, v0);
                if (more) load(k_mine, next, 0, k0);
                put(vst + s * kTile, 1, v1);
                if (more) load(k_mine, next, 1, k1);
                handed(&sm.v_full[s]);
            }
        }
    } else {
        set_registers<false, kRestRegs>();
        if (warp == 13) {
            // --- pages and scales: lanes 8 i .. 8 i + 7 have the 16-key groups of every fourth step from step i on ---
            PrWalk w;
            w.start(a, sm);
            const int g = lane & 7;
            const uint32_t steps = uint32_t(u1 - u0);
            for (uint32_t n0 = 0; n0 < steps; n0 += 4) {
                const uint32_t n = n0 + (lane >> 3);
                float4 sc = make_float4(0.f, 0.f, 1.f, 1.f);
                int64_t codes = -1;
                int from = 0, count = 0;
                if (n < steps) {
                    const int64_t u = u0 + n;
                    w.seek(a, u);
                    const int hk = int((u - w.base) / w.t.steps);
                    const int k0 = w.t.k_begin + int(u - w.base - int64_t(hk) * w.t.steps) * kPrKeys, key = k0 + 16 * g;
                    from = max(w.t.lo - k0, 0), count = max(min(w.t.hi - k0, kPrKeys) - from, 0);
                    if (key + 16 > w.t.lo && key < w.t.hi) {
                        const int page = __ldg(a.table + int64_t(w.b) * a.width + (key >> a.shift));
                        if (page >= 0 && page < a.pages) {
                            const int64_t at = int64_t(page) * Hk + hk;
                            codes = ((at << a.shift) + (key & (P - 1))) * D;
                            const int ve = stored_exponent(__ldg(a.v_scale + at));
                            sc = make_float4(__ldg(a.k_scale + at), float(ve), exp2_int(-ve), 1.f);
                        } else {
                            set_status(a.status, DEV_BAD_INDEX);
                            sc.w = 0.f;
                        }
                    }
                }
                // slot of step n0 + 3: the last of the four to be free
                if (n < steps && n >= kPrSlots)
                    pr_wait(&sm.step_free[n % kPrSlots], (n / kPrSlots - 1) & 1, a.status, abort_flag);
                if (__any_sync(0xffffffffu, *abort_flag)) break;
                if (n < steps) {
                    PrStep& st = sm.step[n % kPrSlots];
                    st.sc[g] = sc;
                    st.at[g] = codes;
                    if (g == 0) st.from = from, st.count = count;
                }
                __syncwarp();
                if (n < steps && g == 0) mbar_arrive(&sm.step_full[n % kPrSlots]);
            }
        }
        if (warp == 14) {
            // --- items ---
            PrWalk w;
            w.start(a, sm);
            int64_t u = u0;
            for (uint32_t it = 0;; ++it) {
                if (it >= kPrItems) pr_wait(&sm.item_free[it % kPrItems], (it / kPrItems - 1) & 1, a.status, abort_flag);
                if (__any_sync(0xffffffffu, *abort_flag)) break;
                PrItem im = {};
                if (u < u1) {
                    w.seek(a, u);
                    im.hk = int((u - w.base) / w.t.steps);
                    im.off = int(u - w.base - int64_t(im.hk) * w.t.steps);
                    im.all = w.t.steps, im.steps = int(min(int64_t(w.t.steps - im.off), u1 - u));
                    im.row0 = w.t.row0, im.col0 = w.t.col0, im.rows = w.t.rows, im.first = w.t.first, im.keys = w.t.keys;
                    im.k_begin = w.t.k_begin;
                    // its first step's place on the line
                    const int64_t first = u - im.off + int64_t(kPrItemCost) * (int64_t(w.index) * Hk + im.hk + 1);
                    im.c0 = int(((first + 1) * ctas - 1) / line), im.c1 = int(((first + im.all) * ctas - 1) / line);
                    u += im.steps;
                }
                if (lane == 0) {
                    sm.item[it % kPrItems] = im;
                    mbar_arrive(&sm.item_full[it % kPrItems]);
                }
                if (im.steps == 0) break;
            }
        }
        if (warp != 12) return;
        // --- the products.  The whole warp runs this, so that addresses stay in uniform registers; an
        // elected lane issues ---
        constexpr uint32_t idesc_s = umma_idesc_f16_f32(128, kPrKeys);
        constexpr uint32_t idesc_o = umma_idesc_f16_f32(128, D) | (1u << 16);  // V: MN-major
        constexpr uint32_t kStep = kTile >> 4;
        const uint64_t qd64 = umma_desc_k_sw128(smem_u32(qs)), vd64 = umma_desc_mn_sw128(smem_u32(vst), kBlk);
        const uint32_t q0 = uint32_t(qd64), k0 = uint32_t(umma_desc_k_sw128(smem_u32(kst))), v0 = uint32_t(vd64);
        const uint32_t hi_k = uint32_t(qd64 >> 32), hi_v = uint32_t(vd64 >> 32);
        auto scores = [&](int t, uint32_t s) {
            const uint32_t qd = q0 + uint32_t(t) * kStep, kd = k0 + s * kStep;
            #pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t at = uint32_t((i >> 2) * kBlk + (i & 3) * 32) >> 4;
                elect_umma_ss(tm + 128 * t, qd + at, kd + at, hi_k, idesc_s, i > 0);
            }
            elect_commit(&sm.s_full[t]);
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            pr_wait(bar, parity, a.status, abort_flag);
            __syncwarp();
        };
        uint32_t n = 0, n1 = 0, items1 = 0;  // steps so far, those with a second tile, items with one
        for (uint32_t items = 0;; ++items) {
            wait(&sm.item_full[items % kPrItems], (items / kPrItems) & 1);
            if (__any_sync(0xffffffffu, *abort_flag)) break;
            const int steps = __shfl_sync(0xffffffffu, sm.item[items % kPrItems].steps, 0);
            const int nt = __shfl_sync(0xffffffffu, sm.item[items % kPrItems].rows, 0) > 128 ? 2 : 1;
            if (steps == 0) break;
            if (lane == 0) mbar_arrive(&sm.item_free[items % kPrItems]);
            __syncwarp();
            wait(&sm.k_full[n & 1], (n >> 1) & 1);
            for (int t = 0; t < nt; ++t) {
                wait(&sm.q_full[t], (t ? items1 : items) & 1);
                tc_fence_after();
                scores(t, n & 1);
            }
            elect_commit(&sm.k_empty[n & 1]);
            items1 += nt - 1;
            for (int j = 0; j < steps; ++j, ++n, n1 += nt - 1) {
                const uint32_t s = n & 1, sn = s ^ 1;
                const bool more = j + 1 < steps;
                if (more) wait(&sm.k_full[sn], ((n + 1) >> 1) & 1);
                wait(&sm.v_full[s], (n >> 1) & 1);
                for (int t = 0; t < nt; ++t) {
                    const uint32_t vd = v0 + s * kStep;
                    wait(&sm.p_full[t], (t ? n1 : n) & 1);
                    tc_fence_after();
                    #pragma unroll
                    for (int i = 0; i < kPrKeys / 16; ++i)
                        elect_umma_ts(tm + 256 + 128 * t, tm + 128 * t + 8 * i, vd + uint32_t(2048 * i >> 4), hi_v, idesc_o,
                                      i > 0 ? 1u : uint32_t(j > 0));
                    elect_commit(&sm.o_full[t]);
                    if (more) scores(t, sn);
                }
                elect_commit(&sm.v_empty[s]);
                if (more) elect_commit(&sm.k_empty[sn]);
            }
        }
        // all products are done, also after a wait that ran out: TMEM and shared memory are free to go
        elect_commit(&sm.done);
        mbar_wait(&sm.done, 0, a.status);
        __syncwarp();
        named_bar_sync(1, 288);  // the rows are read
        tc_fence_after();
        tmem_dealloc(tm, kPrTmem);
    }
}

// One CTA per SM, each with at most two items that it shares with others.
size_t kv_prompt_bytes(const KvAttendCall& c, int sms) { return size_t(sms) * 2 * 2 * 128 * (c.dim + 2) * 4; }

template <bool E4M3, bool BF16, int D>
static cudaError_t launch_prompt(const KvAttendArgs& a, int sms, cudaStream_t s) {
    constexpr size_t smem = pr_smem_bytes<D>();
    static_assert(smem <= 227 * 1024, "shared memory");
    auto* kernel = kv_prompt_kernel<E4M3, BF16, D>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = raise_smem(kernel, smem, done);
    if (e != cudaSuccess) return e;
    kernel<<<sms, kPrThreads, smem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t run_kv_prompt(const KvAttendCall& c, const KvAttendArgs& a, int sms, cudaStream_t s) {
    if (c.requests == 0) return cudaSuccess;
    const auto by_dim = [&](auto e4, auto bf) {
        constexpr bool E = decltype(e4)::value, B = decltype(bf)::value;
        return c.dim == 128 ? launch_prompt<E, B, 128>(a, sms, s) : launch_prompt<E, B, 64>(a, sms, s);
    };
    const bool bf16 = c.x_dtype == DT_BF16;
    if (c.e4m3) return bf16 ? by_dim(std::true_type(), std::true_type()) : by_dim(std::true_type(), std::false_type());
    return bf16 ? by_dim(std::false_type(), std::true_type()) : by_dim(std::false_type(), std::false_type());
}

}  // namespace exl3
