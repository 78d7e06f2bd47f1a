// What the attention kernels share: the packing and mask of a call, a document's span, and the score transforms.
//
// Queries and keys of all documents are packed; document d holds queries cu_q[d] .. cu_q[d+1] and keys cu_k[d] ..
// cu_k[d] + Lk, Lk its own length or, with k_len, the used part of its room.  Query i stands at place p = i + Lk - Lq
// among its document's keys.  It attends to key j where j <= p or j < prefix (causal), or to every key of its document:
// always the keys 0 .. lim of its document, lim = min(Lk - 1, max(p, prefix - 1)), so a row's mask is one number.
//   s = scale q.k;  s = cap tanh(s / cap) where a cap is set;  s = s - slope_h |p - j| where slopes are set.
// Scores are kept in units of log 2 (s2 = s log2 e), so that a probability is one exp2.
#pragma once

#include "tok_common.cuh"

// A whole warp's bounded wait; clears `ok` where any lane gave up.
#define TOK_WAIT(bar, parity)                                                                        \
    do {                                                                                             \
        if (!__all_sync(0xffffffffu, mbar_wait((bar), (parity), abort_flag))) { ok = false; break; } \
    } while (0)

namespace pmg {
namespace tok {

struct Attn {
    const int32_t *cu_q, *cu_k, *k_len, *prefix;
    const float* slopes;
    int64_t Tq, Tk;
    int docs, Hq, Hk, group, D, causal;
    float scale2;            // scale log2 e
    float tanh_in;           // 2 scale log2 e / cap: exp2 of (score * tanh_in) = e^(2 s / cap)
    float cap2;              // cap log2 e
    int32_t* status;
};

struct Span {
    int q0, lq, k0, lk, prefix;      // first query row and count, first key row and count
    int room;                        // key rows that belong to the document
};

// A document's span, cut to the tensors: offsets that leave them, run backwards, or lengths over the room are reported.
__device__ __forceinline__ Span span_of(const Attn& a, int d) {
    Span s;
    s.q0 = min(max(a.cu_q[d], 0), (int)a.Tq);
    s.lq = min(max(a.cu_q[d + 1], s.q0), (int)a.Tq) - s.q0;
    s.k0 = min(max(a.cu_k[d], 0), (int)a.Tk);
    s.room = min(max(a.cu_k[d + 1], s.k0), (int)a.Tk) - s.k0;
    s.lk = a.k_len ? max(0, min(a.k_len[d], s.room)) : s.room;
    if (threadIdx.x == 0 && (s.q0 != a.cu_q[d] || s.q0 + s.lq != a.cu_q[d + 1] || s.k0 != a.cu_k[d] ||
                             s.k0 + s.room != a.cu_k[d + 1] || (a.k_len && s.lk != a.k_len[d])))
        flag(a.status, PMG_ERR_RANGE);
    s.prefix = a.prefix ? min(max(a.prefix[d], 0), s.lk) : 0;
    return s;
}

// The last key that row i (place p = i + lk - lq) sees; negative: none.
__device__ __forceinline__ int last_key(const Attn& a, const Span& s, int i) {
    if (i >= s.lq) return -1;
    return a.causal ? max(i + s.lk - s.lq, s.prefix - 1) : s.lk - 1;
}

// Keys that the rows r0 .. r1 - 1 reach together: 0 .. result - 1.
__device__ __forceinline__ int key_end(const Attn& a, const Span& s, int r1) {
    if (!a.causal) return s.lk;
    return max(0, max(min(r1, s.lq) + s.lk - s.lq, s.prefix));
}

// Document and tile within it of the t-th tile of `rows` rows, counting every document's tiles in order; by one warp.
// false: there are fewer tiles.
__device__ __forceinline__ bool find_tile(const int32_t* cu, int docs, int rows, int t, int* doc, int* tile) {
    const int lane = threadIdx.x & 31;
    for (int d0 = 0; d0 < docs; d0 += 32) {
        const int d = d0 + lane;
        const int n = d < docs ? max(0, cu[d + 1] - cu[d]) : 0, tiles = (n + rows - 1) / rows;
        const int upto = warp_inclusive_scan(tiles);
        const int total = __shfl_sync(0xffffffffu, upto, 31);
        if (t < total) {
            const int l = __ffs(__ballot_sync(0xffffffffu, upto > t)) - 1;
            *doc = d0 + l;
            *tile = t - __shfl_sync(0xffffffffu, upto - tiles, l);
            return true;
        }
        t -= total;
    }
    return false;
}

// cap tanh(s / cap) in units of log 2 from the raw product: cap2 (1 - 2 / (e^(2 s scale / cap) + 1)).  The hardware's
// tanh is off by up to 2^-11, which a cap of 50 would turn into 3 % of a probability; this form is off by about
// 2e-7 cap.
__device__ __forceinline__ float capped(const Attn& a, float s) {
    return fmaf(-2.0f * a.cap2, rcp_approx(ex2(s * a.tanh_in) + 1.0f), a.cap2);
}

}  // namespace tok

// Host: fills an Attn and checks what every attention entry point checks.
int fill_attn(tok::Attn* a, int dtype, const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_len, int docs, int64_t Tq,
              int64_t Tk, int Hq, int Hk, int D, float scale, int causal, const int32_t* prefix, float softcap,
              const float* slopes, int32_t* status);

// Host: tensor map of [T, H, D] with a box of `rows` tokens of one head and 64 values.
int head_map(CUtensorMap* m, const void* p, int64_t tok, int64_t head, int64_t T, int H, int D, int rows);

}  // namespace pmg
