// kv_attend.cuh -- what the two attention kernels over the paged 8-bit cache
// share: their arguments and the conversion of codes to tensor-core operands.
#pragma once

#include "kv_common.cuh"

namespace exl3 {

// A column's weights are taken against a reference that starts this far (log2)
// below its maximum, and follows it when it has grown by kAttSlack more: the
// largest weight is 2^7 to 2^15, so that f16 holds weights down to 2^-21 of it in
// full and down to 2^-32 at all.  (Against the maximum itself those ends are
// 2^-14 and 2^-25: behind one key that takes all the weight, a long tail 17 nats
// below it came out 41 % too large, or as nothing.)  The sums l, fp32, are
// taken against the same reference.
constexpr float kAttLift = 7.f, kAttSlack = 8.f;

struct KvAttendArgs {
    const uint16_t* q;
    int64_t q_tok, q_head, q_rows;
    int heads, kv_heads, group;  // group = heads / kv_heads
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    int64_t pages;
    int shift;
    const int32_t* table;
    int width, requests;
    const int32_t *kv_lens, *cu;
    float scale_log2;  // softmax scale * log2(e)
    int window;
    int few;  // requests of more query columns (rows x group) than this are the prompt kernel's
    uint16_t* out;
    float* lse;
    int32_t* counters;
    float* part;
    int* status;
};

// A request's rows of q: its positions count from all `fresh` that cu_tokens
// names, `rows` of them are computed.  They are fewer where cu_tokens leaves
// the tensor, so that no offset here leaves it.
struct AttRows {
    int row0, fresh, rows;
};
__device__ __forceinline__ AttRows att_rows(const KvAttendArgs& a, int b) {
    if (!a.cu) return AttRows{b, 1, 1};
    const int row0 = a.cu[b], end = a.cu[b + 1];
    const int n = row0 >= 0 && end > row0 ? end - row0 : 0;
    return AttRows{row0, n, min(n, max(int(a.q_rows) - row0, 0))};
}

// Tokens of a request that the block table has a place for.  The others are
// not seen; they count for the rows' positions all the same.
__device__ __forceinline__ int att_keys(const KvAttendArgs& a, int len) { return min(len, a.width << a.shift); }

// Records a request whose rows leave q or whose tokens leave the table
__device__ __forceinline__ void att_check(const KvAttendArgs& a, int b) {
    const AttRows w = att_rows(a, b);
    const bool before = a.cu && a.cu[b] < 0 && a.cu[b + 1] > a.cu[b];
    if (before || w.rows < w.fresh || a.kv_lens[b] > a.width << a.shift) set_status(a.status, DEV_BAD_INDEX);
}

// two codes (bytes 0, 1 of w; int8 already offset by 128) as f16x2, exact
template <bool E4M3>
__device__ __forceinline__ uint32_t half2_lo(uint32_t w) {
    if constexpr (E4M3) {
        return e4m3x2_lo(w);
    } else {
        uint32_t h = __byte_perm(w, 0x64646464u, 0x4140);  // 1024 + u
        const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), __float2half2_rn(1152.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t half2_hi(uint32_t w) {
    if constexpr (E4M3) {
        return e4m3x2_hi(w);
    } else {
        uint32_t h = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), __float2half2_rn(1152.f));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t code_word(uint32_t w) {
    return E4M3 ? w : w ^ 0x80808080u;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// kv_prompt.cu: requests with more than `few` query columns
size_t kv_prompt_bytes(const KvAttendCall& c, int sms);  // of its partial results
cudaError_t run_kv_prompt(const KvAttendCall& c, const KvAttendArgs& a, int sms, cudaStream_t s);

}  // namespace exl3
