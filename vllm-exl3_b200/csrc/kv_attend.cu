// kv_attend.cu -- attention over the paged 8-bit cache, few query rows per request.
//
//   out[r] = sum_j softmax_j(scale * q_r . k_j) v_j over the keys j that row r
//   may see: j <= pos_r, j < len, and j > pos_r - window where there is a window.
//
// The scales of a (page, head) tile are constant over it, so with e = log2 of
// the V scale the tile's weights are p_j = 2^(s_j + e - m), m the running
// maximum of s_j + e, and
//   out = sum_j p_j code_j / sum_j p_j 2^-e :
// codes feed the tensor core as they are and no value is multiplied by a scale.
//
// Work: an item is (request, kv head, group of NC = 8 NT query columns), a
// column being one (token, query head) that reads this kv head.  Its keys are
// cut into units of 128 (8 warps x 16 keys); all items' units, and a few for
// each item's start and end, form one line that the CTAs split evenly, so
// lengths need no balancing and the host needs none of them.  An item cut by a CTA boundary is joined from fp32 partials by
// the CTA that finishes it last, in key order (results do not depend on timing).
//
// Bound: every code is read once, 2 D bytes per (key, kv head): HBM.  Each
// warp copies its own 16-key tiles into a ring of its own in shared memory
// (cp.async, 16 bytes a lane), two or more tiles ahead: some 128 KB in flight
// per SM and no CTA barrier inside the loop.  The tiles are swizzled (16-byte
// chunk ^= row mod 8) so that the fragments' 16-byte loads are free of bank
// conflicts.  The products run as S^T = K Q^T and O^T = V^T P^T on m16n8k16:
// the keys (then the dims) are the 16 rows, so 8 query columns fill an MMA.  A
// dim may sit at any place of the contraction, so a lane's 16 bytes already
// are its A fragment of K; for V, words of two keys are interleaved with one
// byte permute.  Like the prompt kernel, a column's reference follows its
// maximum only when that has grown by more than 2^8 (kAttSlack), so that the usual
// tile needs no exchange between lanes and no rescaling.
//
// Measured (lone calls): 64 single tokens over up to 8192 keys (32 heads over 4,
// dim 128, e4m3, 343 MB) 69 us, 4.95 TB/s, 76 % of the measured copy rate; 4
// requests of 3 tokens over up to 128K keys (64 heads over 8, int8, 24 columns)
// 212 us, 59 % (the int8 conversions and three column tiles leave two warps per
// scheduler at their issue latency); one token over 1021 keys 11.2 us, 9.9 in a
// graph, a chain of dependent steps.  A piece of an item costs about 13K cycles
// beside its tiles (queries in, warps joined, partials out), a third of a CTA's
// time at the 64.  The request's numbers stay in shared memory over the loop:
// in registers they took 71, 220 and 12.3 us.
// Not kept, us at the 64 and the 128K: joining at a CTA's end 77 / 250, joining
// the warps as a tree 76 / 233, separate loops for tiles with and without masks 74 / 217
// (each against 71 / 218 then).
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "kv_attend.cuh"

namespace exl3 {

constexpr int kAttWarps = 8, kAttThreads = kAttWarps * 32, kAttUnit = 16 * kAttWarps;
constexpr int kAttMaxSms = 160;     // SMs that are used at most
// Units that an item's start and end are worth on the line, where the CTAs have more than a unit each.  us with 0 / 3 / 5 / 10:
//   64 single tokens over up to 8192 keys (32 heads over 4, e4m3) 71.4 / 69.5 / 70.0 / 71.6
//   25 x 4 tokens, 20918 keys (12 heads over 4, int8) 102.6 / 99.7 / 95.9 / 98.3
//   dim 64, int8: 126 single tokens, 2309 keys (12 heads over 1) 24.7 / 22.7 / 21.5 / 22.7, 127, 697 keys (8 over 2) 20.6 / 16.6 / 17.4 / 16.5
//   4 x 3 tokens over 128K keys (24 columns) 216.6 / 221.5 / 218.0 / 220.0
constexpr int kAttItemCost = 5;

// Tiles of 8 query columns an item has at most: up to two with two CTAs per
// SM; three or four need the registers of one.
template <int D, int NT>
struct AttShape {
    static constexpr int NC = 8 * NT;
    static constexpr int kCtas = NT <= 2 ? 2 : 1;
    static constexpr int kTile = 16 * D;                          // bytes of 16 keys of K, or of V
    static constexpr int kStages = (NT <= 2 ? 3 : 6) * 128 / D;   // 96 KB of ring per CTA, 192 KB where it is alone
    static constexpr int kRing = kAttWarps * kStages * 2 * kTile;
    static constexpr int kRed = kAttWarps * NC * D * 4;           // the warps' outputs take the ring's place
    // the ring holds the join of the warps, and that of the pieces: one per CTA at most, of up to kAttMaxSms SMs
    static_assert(kRed <= kRing && kAttMaxSms * kCtas * 2 * NC * 4 <= kRing, "the joins fit the ring");
    static constexpr int kQ = NT * (D / 16) * 32 * 8;             // Q fragments
    static constexpr int kSmem = kRing + kQ + (2 * kAttWarps * NC + 3 * NC) * 4 + kAttWarps * kStages * 8;
};

// Requests of more query columns (rows x heads per kv head) than this go to
// the prompt kernel when the call has such requests at all.  From 33 on the
// kernel here reads the keys twice (the second time from L2), the prompt kernel
// pads to 128 rows.  us here / there, int8, dim 128, 64 heads over 8:
//   8 requests of 32K keys: 24 columns 111 / 186, 32 142 / 237, 40 159 / 213, 48 189 / 222, 64 225 / 225, 96 271 / 223
//   64 requests of 1K keys: 24 88 / 112, 32 104 / 111, 40 111 / 96, 64 159 / 98
constexpr int kAttFew = 48;

// what a request asks for
struct AttReq {
    int keys, first, rows, lo16, groups, units;  // keys, first row's position, rows, first key's tile, column groups, units per item
    int64_t row0;
};

template <int NC>
__device__ __forceinline__ AttReq att_request(const KvAttendArgs& a, int b) {
    AttReq r;
    const AttRows w = att_rows(a, b);
    r.row0 = w.row0, r.rows = w.rows;
    const int len = max(a.kv_lens[b], 0);
    r.keys = att_keys(a, len), r.first = len - w.fresh;
    const int lo = a.window > 0 ? max(r.first + 1 - a.window, 0) : 0;
    r.lo16 = min(lo, r.keys) & ~15;
    const int64_t columns = int64_t(r.rows) * a.group;
    r.groups = columns > a.few ? 0 : int((columns + NC - 1) / NC);
    r.units = max((r.keys - r.lo16 + kAttUnit - 1) / kAttUnit, 1);
    return r;
}

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

template <bool E4M3, bool BF16, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, (AttShape<D, NT>::kCtas)) kv_attend_kernel(const KvAttendArgs a) {
    using Shape = AttShape<D, NT>;
    constexpr int NC = 8 * NT;
    constexpr int KS = D / 16;  // contraction steps of S, row tiles of O
    constexpr int PART = NC * (D + 2);
    constexpr int S = Shape::kStages;
    constexpr bool kQRegs = NT == 1;                  // Q fragments in registers, else read from shared memory
    extern __shared__ __align__(128) char att_smem[];
    float* red = reinterpret_cast<float*>(att_smem);  // [warps][NC][D], in the ring's place
    uint2* qs = reinterpret_cast<uint2*>(att_smem + Shape::kRing);                    // [NT][KS][32]
    float* wm = reinterpret_cast<float*>(att_smem + Shape::kRing + Shape::kQ);        // [warps][NC] maxima, then factors
    float* wl = wm + kAttWarps * NC;                  // [warps][NC] sums
    float* fin = wl + kAttWarps * NC;                 // [2][NC] joined maximum, sum
    float* qfac = fin + 2 * NC;                       // [NC] factor of a column's scores
    float2* tile_sc = reinterpret_cast<float2*>(qfac + NC);  // [warps][S] a tile's K and V scale
    __shared__ int64_t scan[2][kAttWarps];
    __shared__ int64_t found_base;
    __shared__ AttReq found;
    __shared__ int found_b, last_flag;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int Hk = a.kv_heads, G = a.group, P = 1 << a.shift;

    // --- this CTA's share of the line of units ---
    const int per = (a.requests + kAttThreads - 1) / kAttThreads;
    int64_t mine = 0, items = 0;
    AttReq own = {};
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        if (b < a.requests) {
            own = att_request<NC>(a, b);
            if (blockIdx.x == 0) att_check(a, b);  // of every request, the prompt kernel's too
            mine += int64_t(own.groups) * Hk * own.units;
            items += int64_t(own.groups) * Hk;
        }
    }
    int64_t incl = mine, items_incl = items;
    #pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, incl, d), oi = __shfl_up_sync(0xffffffffu, items_incl, d);
        if (lane >= d) incl += o, items_incl += oi;
    }
    if (lane == 31) scan[0][warp] = incl, scan[1][warp] = items_incl;
    __syncthreads();
    int64_t total = 0, n_items = 0;
    #pragma unroll
    for (int w = 0; w < kAttWarps; ++w) {
        if (w == warp) incl += total, items_incl += n_items;
        total += scan[0][w], n_items += scan[1][w];
    }
    // an item's line: `cost` places, then its units
    const int cost = total > gridDim.x ? kAttItemCost : 0;
    total += cost * n_items, incl += cost * items_incl, mine += cost * items;
    // rows no request owns are zeros
    if (a.cu) {
        const int64_t live = max(a.cu[a.requests], 0), n = (a.q_rows - live) * a.heads;
        for (int64_t i = int64_t(blockIdx.x) * kAttWarps + warp; i < n; i += int64_t(gridDim.x) * kAttWarps) {
            const int64_t row = live * a.heads + i;
            for (int d = lane; d < D; d += 32) a.out[row * D + d] = 0;
            if (a.lse && lane == 0) a.lse[row] = -INFINITY;
        }
    }
    const int ctas = int(min(int64_t(gridDim.x), total));
    const int cta = blockIdx.x;
    if (cta >= ctas) return;
    int64_t u = total * cta / ctas;
    const int64_t u_end = total * (cta + 1) / ctas;
    if (u >= incl - mine && u < incl) {
        int64_t base = incl - mine;
        int b = tid * per;
        for (;;) {
            const AttReq r = per == 1 ? own : att_request<NC>(a, b);
            const int64_t n = int64_t(r.groups) * Hk * (r.units + cost);
            if (u < base + n) {
                found = r;
                break;
            }
            base += n, ++b;
        }
        found_b = b, found_base = base;
    }
    __syncthreads();
    int b = found_b;
    int64_t base = found_base;
    AttReq rq = found;

    while (u < u_end) {
        while (u >= base + int64_t(rq.groups) * Hk * (rq.units + cost)) {  // next request with work
            base += int64_t(rq.groups) * Hk * (rq.units + cost);
            rq = att_request<NC>(a, ++b);
            if (tid == 0) found = rq;
        }
        const int64_t item = (u - base) / (rq.units + cost), u_item = base + item * (rq.units + cost) + cost;  // its first unit
        const int off = int(max(u - u_item, int64_t(0)));
        u = min(u_item + rq.units, u_end);
        const int n_units = int(u - u_item) - off;
        if (n_units <= 0) break;  // the CTA's part of the line ends before the item's first unit
        const int hk = int(item / rq.groups), cg = int(item % rq.groups);
        const int ncols = int(min(int64_t(rq.rows) * G - int64_t(cg) * NC, int64_t(NC)));

        // --- the query columns: B fragments of Q^T (a warp to each 8), and each column's key range ---
        for (int t = warp; t < NT; t += kAttWarps) {
            const int n = 8 * t + g, f = cg * NC + n;
            const int64_t row = rq.row0 + f / G;
            const bool live = n < ncols;
            const uint16_t* qp = a.q + (live ? row * a.q_tok + int64_t(hk * G + f % G) * a.q_head : 0);
            float fac = a.scale_log2;
            uint2 w[KS];
            #pragma unroll
            for (int s = 0; s < KS; ++s) {
                // contraction step s takes word s % 4 of this lane's chunk of K
                const int dim = (D == 128 ? (2 * c + (s >> 2)) * 16 : c * 16) + (s & 3) * 4;
                w[s] = live ? *reinterpret_cast<const uint2*>(qp + dim) : make_uint2(0u, 0u);
            }
            if constexpr (BF16) {
                // the tensor core takes Q in f16 like the codes: a power of two per row puts its
                // largest magnitude in [2^14, 2^15), where f16 keeps all 8 bits of a bf16 value
                // down to 2^-31 of that largest one
                uint32_t m2 = 0;
                #pragma unroll
                for (int s = 0; s < KS; ++s) m2 = __vmaxu2(m2, __vmaxu2(w[s].x & 0x7fff7fffu, w[s].y & 0x7fff7fffu));
                float amax = fmaxf(__uint_as_float(m2 << 16), __uint_as_float(m2 & 0xffff0000u));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int e = min(max((__float_as_int(amax) >> 23) - 127, -100), 100);
                const float mul = exp2_int(14 - e);
                fac *= exp2_int(e - 14);
                auto conv = [&](uint32_t v) { return pack_half2(__uint_as_float(v << 16) * mul, __uint_as_float(v & 0xffff0000u) * mul); };
                #pragma unroll
                for (int s = 0; s < KS; ++s) w[s] = make_uint2(conv(w[s].x), conv(w[s].y));
            }
            #pragma unroll
            for (int s = 0; s < KS; ++s) qs[(t * KS + s) * 32 + lane] = w[s];
            if (c == 0) qfac[8 * t + g] = fac;
        }
        __syncthreads();
        uint2 qf[kQRegs ? NT : 1][KS];
        if constexpr (kQRegs) {
            #pragma unroll
            for (int t = 0; t < NT; ++t)
                #pragma unroll
                for (int s = 0; s < KS; ++s) qf[t][s] = qs[(t * KS + s) * 32 + lane];
        }
        float cfac[NT][2];           // columns 2c, 2c + 1
        int hi[NT][2], lo[NT][2];    // keys [lo, hi)
        #pragma unroll
        for (int t = 0; t < NT; ++t)
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int col = 8 * t + 2 * c + i, pos = rq.first + (cg * NC + col) / G;
                cfac[t][i] = qfac[col];
                hi[t][i] = col < ncols ? min(pos + 1, rq.keys) : 0;
                lo[t][i] = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
            }
        int full_lo = 0, full_hi = 0x7fffffff;  // keys in [full_lo, full_hi) need no test
        #pragma unroll
        for (int t = 0; t < NT; ++t)
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool live = 8 * t + 2 * c + i < ncols;
                full_lo = max(full_lo, live ? lo[t][i] : 0);
                full_hi = min(full_hi, live ? hi[t][i] : 0x7fffffff);
            }
        full_lo = __reduce_max_sync(0xffffffffu, full_lo);
        full_hi = __reduce_min_sync(0xffffffffu, full_hi);

        float o[NT][KS][4], m[NT][2], l[NT][2];
        #pragma unroll
        for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int j = 0; j < KS; ++j)
                #pragma unroll
                for (int i = 0; i < 4; ++i) o[t][j][i] = 0.f;
            m[t][0] = m[t][1] = -INFINITY;
            l[t][0] = l[t][1] = 0.f;
        }

        const int first = rq.lo16 + off * kAttUnit + warp * 16;
        const int end = min(rq.keys, rq.lo16 + (off + n_units) * kAttUnit);
        const int32_t* row_table = a.table + int64_t(b) * a.width;
        auto page_at = [&](int tok) { return tok < end ? __ldg(row_table + (tok >> a.shift)) : -1; };

        const uint32_t ring = smem_u32(att_smem) + warp * (S * 2 * Shape::kTile);
        const uint32_t ring_sc = smem_u32(tile_sc) + warp * (S * 8);
        // where chunk lane (+ 32, + 64, ...) of a tile goes: 16-byte chunk ^= row mod 8 (rows of 64 bytes: row / 2 mod 4)
        constexpr int CH = D / 16;
        const int cr = lane / CH, cc = lane % CH;
        auto fetch = [&](int tok, int page, int stage) {
            const bool get = tok < end && page >= 0 && page < a.pages;
            if (get) {
                const int64_t tile = int64_t(page) * Hk + hk;
                const int64_t at = ((tile << a.shift) + (tok & (P - 1))) * D + lane * 16;
                const uint32_t dst = ring + stage * (2 * Shape::kTile);
                #pragma unroll
                for (int i = 0; i < CH / 2; ++i) {
                    const int row = cr + i * (32 / CH);
                    const uint32_t to = dst + row * D + ((cc ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4);
                    copy_async16(to, a.k + at + i * 512);
                    copy_async16(to + Shape::kTile, a.v + at + i * 512);
                }
                if (lane < 2) copy_async4(ring_sc + stage * 8 + lane * 4, (lane ? a.v_scale : a.k_scale) + tile);
            } else if (tok < end && lane == 0) {
                set_status(a.status, DEV_BAD_INDEX);
            }
            copy_commit();
            return get;
        };
        // this warp's tiles: first, first + kAttUnit, ...; S - 1 of them are on their way
        uint32_t have = 0;  // bit i: tile (present + i) exists
        {
            int ahead[S - 1];
            #pragma unroll
            for (int i = 0; i < S - 1; ++i) ahead[i] = page_at(first + i * kAttUnit);
            #pragma unroll
            for (int i = 0; i < S - 1; ++i) have |= uint32_t(fetch(first + i * kAttUnit, ahead[i], i)) << i;
        }
        int page_next = page_at(first + (S - 1) * kAttUnit);
        int stage = 0;
        for (int tok = first; tok < end; tok += kAttUnit) {
            copy_wait<S - 2>();
            __syncwarp();  // the tile is here, for all lanes, and the one before it is done with
            {
                const int page = page_next, t = tok + (S - 1) * kAttUnit;
                page_next = page_at(t + kAttUnit);
                have |= uint32_t(fetch(t, page, stage == 0 ? S - 1 : stage - 1)) << (S - 1);
            }
            const bool here = have & 1u;
            have >>= 1;
            const char* kt = att_smem + warp * (S * 2 * Shape::kTile) + stage * (2 * Shape::kTile);
            const char* vt = kt + Shape::kTile;
            const float2 sc = tile_sc[warp * S + stage];
            stage = stage == S - 1 ? 0 : stage + 1;
            if (!here) continue;

            // --- S^T = K Q^T: keys g and g + 8 ---
            float s[NT][4];
            #pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
            #pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                const int sw = D == 128 ? ((2 * c + h) ^ (g & 7)) << 4 : (c ^ ((g >> 1) & 3)) << 4;
                const uint4 x = *reinterpret_cast<const uint4*>(kt + g * D + sw);
                const uint4 y = *reinterpret_cast<const uint4*>(kt + (g + 8) * D + sw);
                #pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t w0 = code_word<E4M3>(q == 0 ? x.x : q == 1 ? x.y : q == 2 ? x.z : x.w);
                    const uint32_t w1 = code_word<E4M3>(q == 0 ? y.x : q == 1 ? y.y : q == 2 ? y.z : y.w);
                    const uint32_t af[4] = {half2_lo<E4M3>(w0), half2_lo<E4M3>(w1), half2_hi<E4M3>(w0), half2_hi<E4M3>(w1)};
                    #pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint2 bq = kQRegs ? qf[kQRegs ? t : 0][4 * h + q] : qs[(t * KS + 4 * h + q) * 32 + lane];
                        mma_16816(s[t], af, bq.x, bq.y);
                    }
                }
            }
            // V: keys 2c, 2c + 1, 2c + 8, 2c + 9, dims g * D / 8 and on
            uint32_t vr[4][D / 32];
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 2 * c + (i & 1) + (i >> 1) * 8;
                if constexpr (D == 128) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vt + row * D + ((g ^ (row & 7)) << 4));
                    vr[i][0] = w.x, vr[i][1] = w.y, vr[i][2] = w.z, vr[i][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(vt + row * D + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
                    vr[i][0] = w.x, vr[i][1] = w.y;
                }
            }

            // --- weights of these 16 keys ---
            const int ve = stored_exponent(sc.y);
            const float vexp = float(ve), vinv = exp2_int(-ve);
            const bool edge = tok < full_lo || tok + 16 > full_hi;
            bool grown = false;
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) s[t][i] = fmaf(s[t][i], cfac[t][i & 1] * sc.x, vexp);
                if (edge) {
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = tok + g + 8 * (i >> 1);
                        if (key >= hi[t][i & 1] || key < lo[t][i & 1]) s[t][i] = -INFINITY;
                    }
                }
                #pragma unroll
                for (int i = 0; i < 2; ++i) grown |= fmaxf(s[t][i], s[t][i + 2]) > m[t][i] + (kAttLift + kAttSlack);
            }
            if (__any_sync(0xffffffffu, grown)) {  // -inf + slack is -inf: the first key that is seen counts as growth
                #pragma unroll
                for (int t = 0; t < NT; ++t)
                    #pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float mx = fmaxf(m[t][i], fmaxf(s[t][i], s[t][i + 2]) - kAttLift);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float alpha = mx == m[t][i] ? 1.f : ex2(m[t][i] - mx);  // 0 where nothing has been seen
                        m[t][i] = mx;
                        l[t][i] *= alpha;
                        #pragma unroll
                        for (int j = 0; j < KS; ++j) o[t][j][i] *= alpha, o[t][j][i + 2] *= alpha;
                    }
            }
            uint32_t pf[NT][2];
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
                float p[4];
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ref = m[t][i] == -INFINITY ? 0.f : m[t][i];
                    p[i] = ex2(s[t][i] - ref), p[i + 2] = ex2(s[t][i + 2] - ref);
                    l[t][i] = fmaf(p[i] + p[i + 2], vinv, l[t][i]);
                }
                pf[t][0] = transpose8x8(pack_half2(p[0], p[1]));
                pf[t][1] = transpose8x8(pack_half2(p[2], p[3]));
            }
            if (E4M3 && tok + 16 > rq.keys) {  // codes past the end may be NaN, and 0 * NaN is not 0
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok + 2 * c + (i & 1) + (i >> 1) * 8 >= rq.keys)
                        #pragma unroll
                        for (int w = 0; w < D / 32; ++w) vr[i][w] = 0u;
            }

            // --- O^T += V^T P^T ---
            #pragma unroll
            for (int w = 0; w < D / 32; ++w) {
                const uint32_t v0 = code_word<E4M3>(vr[0][w]), v1 = code_word<E4M3>(vr[1][w]);
                const uint32_t v2 = code_word<E4M3>(vr[2][w]), v3 = code_word<E4M3>(vr[3][w]);
                #pragma unroll
                for (int h = 0; h < 2; ++h) {  // dims 4w + 2h, 4w + 2h + 1 of the lane's D / 8
                    const uint32_t x = __byte_perm(v0, v1, h ? 0x7362 : 0x5140);
                    const uint32_t y = __byte_perm(v2, v3, h ? 0x7362 : 0x5140);
                    const uint32_t af[4] = {half2_lo<E4M3>(x), half2_hi<E4M3>(x), half2_lo<E4M3>(y), half2_hi<E4M3>(y)};
                    #pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16816(o[t][2 * w + h], af, pf[t][0], pf[t][1]);
                }
            }
        }
        copy_wait<0>();
        __syncthreads();  // the ring is free
        rq = found;       // its registers were the loop's

        // --- join the warps ---
        #pragma unroll
        for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], d);
                if (g == 0) wm[warp * NC + 8 * t + 2 * c + i] = m[t][i], wl[warp * NC + 8 * t + 2 * c + i] = l[t][i];
                #pragma unroll
                for (int j = 0; j < KS; ++j)
                    *reinterpret_cast<float2*>(red + (warp * NC + 8 * t + 2 * c + i) * D + g * (D / 8) + 2 * j) =
                        make_float2(o[t][j][i], o[t][j][i + 2]);
            }
        }
        __syncthreads();
        if (tid < NC) {
            float mx = -INFINITY, sum = 0.f;
            for (int w = 0; w < kAttWarps; ++w) mx = fmaxf(mx, wm[w * NC + tid]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            for (int w = 0; w < kAttWarps; ++w) {
                const float f = ex2(wm[w * NC + tid] - ref);
                wm[w * NC + tid] = f;
                sum = fmaf(wl[w * NC + tid], f, sum);
            }
            fin[tid] = mx, fin[NC + tid] = sum;
        }
        __syncthreads();
        auto emit = [&](int col, int d, float value, float sum, float mx) {
            const int f = cg * NC + col;
            const int64_t row = rq.row0 + f / G;
            if (col >= ncols) return;
            const int64_t at = row * a.heads + hk * G + f % G;
            const float r = sum == 0.f ? 0.f : value / sum;  // a row that sees no key is zero
            a.out[at * D + d] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(r)) : __half_as_ushort(__float2half_rn(r));
            if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.6931471805599453f;
        };
        const bool whole = n_units == rq.units;
        // partial slots: 2 cta + 1 for the item that begins in this CTA, 2 cta for the one it carries on
        float* part = a.part + int64_t(2 * cta + (off == 0 ? 1 : 0)) * PART;
        for (int i = tid; i < NC * D; i += kAttThreads) {
            const int col = i / D, d = i % D;
            float v = 0.f;
            #pragma unroll
            for (int w = 0; w < kAttWarps; ++w) v = fmaf(red[(w * NC + col) * D + d], wm[w * NC + col], v);
            if (whole) emit(col, d, v, fin[NC + col], fin[col]);
            else __stcg(part + 2 * NC + i, v);
        }
        if (!whole) {
            if (tid < 2 * NC) __stcg(part + tid, fin[tid]);
            const int64_t T = total;
            const int c0 = int(((u_item + 1) * ctas - 1) / T), c1 = int(((u_item + rq.units) * ctas - 1) / T);
            const int pieces = c1 - c0 + 1;
            __syncthreads();
            if (tid == 0) {
                int prev;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(prev) : "l"(a.counters + c0) : "memory");
                last_flag = prev == pieces - 1;
                if (prev == pieces - 1) a.counters[c0] = 0;  // ready for the next call
            }
            __syncthreads();
            if (last_flag) {
                auto piece = [&](int p) { return a.part + int64_t(2 * (c0 + p) + (p == 0 ? 1 : 0)) * PART; };
                float* wt = red;                   // [pieces][NC] maxima, then weights
                float* wsum = red + pieces * NC;   // [pieces][NC] sums
                for (int i = tid; i < pieces * NC; i += kAttThreads) {
                    const float* pc = piece(i / NC);
                    wt[i] = __ldcg(pc + i % NC), wsum[i] = __ldcg(pc + NC + i % NC);
                }
                __syncthreads();
                if (tid < NC) {
                    float mx = -INFINITY, sum = 0.f;
                    for (int p = 0; p < pieces; ++p) mx = fmaxf(mx, wt[p * NC + tid]);
                    const float ref = mx == -INFINITY ? 0.f : mx;
                    for (int p = 0; p < pieces; ++p) {
                        const float f = ex2(wt[p * NC + tid] - ref);
                        wt[p * NC + tid] = f;
                        sum = fmaf(wsum[p * NC + tid], f, sum);
                    }
                    fin[tid] = mx, fin[NC + tid] = sum;
                }
                __syncthreads();
                for (int i = tid; i < NC * D; i += kAttThreads) {
                    const int col = i / D;
                    float v = 0.f;
                    #pragma unroll 8
                    for (int p = 0; p < pieces; ++p) v = fmaf(__ldcg(piece(p) + 2 * NC + i), wt[p * NC + col], v);
                    emit(col, i % D, v, fin[NC + col], fin[col]);
                }
            }
        }
        __syncthreads();  // shared memory is the next item's
    }
}

// counters: one per CTA of the kernel here, two per CTA of the prompt kernel
int kv_attend_counters(int sms) { return sms * 4; }

static int64_t att_columns(const KvAttendCall& c) { return int64_t(c.max_new) * (c.heads / c.kv_heads); }
static int att_tiles(const KvAttendCall& c) {
    const int64_t n = (att_columns(c) + 7) / 8;
    return int(n < 4 ? n : 4);
}
static size_t att_bytes(const KvAttendCall& c, int sms) {
    const int nt = att_tiles(c);
    return size_t(sms) * (nt <= 2 ? 2 : 1) * 2 * (8 * nt) * (c.dim + 2) * 4;
}

size_t kv_attend_workspace(const KvAttendCall& c, int sms) {
    return att_bytes(c, sms) + (att_columns(c) > kAttFew ? kv_prompt_bytes(c, sms) : 0);
}

template <bool E4M3, bool BF16, int D, int NT>
static cudaError_t launch_attend(const KvAttendArgs& a, int sms, cudaStream_t s) {
    using Shape = AttShape<D, NT>;
    auto* kernel = kv_attend_kernel<E4M3, BF16, D, NT>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = raise_smem(kernel, Shape::kSmem, done);
    if (e != cudaSuccess) return e;
    kernel<<<(sms < kAttMaxSms ? sms : kAttMaxSms) * Shape::kCtas, kAttThreads, Shape::kSmem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t run_kv_attend(const KvAttendCall& c, int sms, cudaStream_t s) {
    if (c.q_rows <= 0) return cudaSuccess;
    KvAttendArgs a;
    a.q = static_cast<const uint16_t*>(c.q), a.q_tok = c.q_tok, a.q_head = c.q_head, a.q_rows = c.q_rows;
    a.heads = c.heads, a.kv_heads = c.kv_heads, a.group = c.heads / c.kv_heads;
    a.k = static_cast<const uint8_t*>(c.k), a.v = static_cast<const uint8_t*>(c.v);
    a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.pages = c.pages, a.shift = page_shift(c.page);
    a.table = c.table, a.width = c.width, a.requests = c.requests, a.kv_lens = c.kv_lens, a.cu = c.cu;
    a.scale_log2 = c.scale * 1.4426950408889634f, a.window = c.window;
    a.out = static_cast<uint16_t*>(c.out), a.lse = c.lse, a.counters = c.counters;
    a.part = reinterpret_cast<float*>(c.ws), a.status = c.status;
    a.few = INT32_MAX;
    if (att_columns(c) > kAttFew) {
        a.few = kAttFew;
        KvAttendArgs p = a;
        p.counters = c.counters + sms * 2;
        p.part = reinterpret_cast<float*>(c.ws + att_bytes(c, sms));
        const cudaError_t e = run_kv_prompt(c, p, sms, s);
        if (e != cudaSuccess) return e;
    }
    const bool bf16 = c.x_dtype == DT_BF16, d128 = c.dim == 128;
    const int nt = att_tiles(c);
    const auto pick = [&](auto e4, auto bf, auto dim) {
        constexpr bool E = decltype(e4)::value, B = decltype(bf)::value;
        constexpr int Dm = decltype(dim)::value;
        return nt == 1   ? launch_attend<E, B, Dm, 1>(a, sms, s)
               : nt == 2 ? launch_attend<E, B, Dm, 2>(a, sms, s)
               : nt == 3 ? launch_attend<E, B, Dm, 3>(a, sms, s)
                         : launch_attend<E, B, Dm, 4>(a, sms, s);
    };
    const auto by_dim = [&](auto e4, auto bf) {
        return d128 ? pick(e4, bf, std::integral_constant<int, 128>()) : pick(e4, bf, std::integral_constant<int, 64>());
    };
    if (c.e4m3) return bf16 ? by_dim(std::true_type(), std::true_type()) : by_dim(std::true_type(), std::false_type());
    return bf16 ? by_dim(std::false_type(), std::true_type()) : by_dim(std::false_type(), std::false_type());
}

}  // namespace exl3
