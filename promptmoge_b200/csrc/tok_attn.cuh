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
        if (!__all_sync(0xffffffffu, wait_bar((bar), (parity), abort_flag))) { ok = false; break; } \
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
    float cap_in;            // scale / cap
    int32_t* status;
};

struct Span {
    int q0, lq, k0, lk, prefix;      // first query row and count, first key row and count
    int room;                        // key rows that belong to the document
};

// A document's span, cut to the tensors: offsets that leave them, run backwards, or lengths over the room.
__device__ __forceinline__ Span cut_span(const Attn& a, int d, bool* bad) {
    Span s;
    s.q0 = min(max(a.cu_q[d], 0), (int)a.Tq);
    s.lq = min(max(a.cu_q[d + 1], s.q0), (int)a.Tq) - s.q0;
    s.k0 = min(max(a.cu_k[d], 0), (int)a.Tk);
    s.room = min(max(a.cu_k[d + 1], s.k0), (int)a.Tk) - s.k0;
    s.lk = a.k_len ? max(0, min(a.k_len[d], s.room)) : s.room;
    *bad = s.q0 != a.cu_q[d] || s.q0 + s.lq != a.cu_q[d + 1] || s.k0 != a.cu_k[d] || s.k0 + s.room != a.cu_k[d + 1] ||
           (a.k_len && s.lk != a.k_len[d]);
    s.prefix = a.prefix ? min(max(a.prefix[d], 0), s.lk) : 0;
    return s;
}
__device__ __forceinline__ Span span_of(const Attn& a, int d) {
    bool bad;
    return cut_span(a, d, &bad);
}

// Reports a document whose span had to be cut, or that has more than max_q queries.
__device__ __forceinline__ void report_span(const Attn& a, int d, int max_q) {
    bool bad;
    const Span s = cut_span(a, d, &bad);
    if (bad || s.lq > max_q) flag(a.status, PMG_ERR_RANGE);
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

// The same tiles level by level: the first tile of every document, then the second of those that have one, and so on.  A
// causal document's tiles shrink from one end to the other; taken in this order from that end, what a GPU starts last is
// small, whatever document it belongs to.
__device__ __forceinline__ bool find_level(const int32_t* cu, int docs, int rows, int t, int* doc, int* level) {
    const int lane = threadIdx.x & 31;
    for (int e = 0;; ++e) {
        int found = 0;
        for (int d0 = 0; d0 < docs; d0 += 32) {
            const int d = d0 + lane;
            const int n = d < docs ? max(0, cu[d + 1] - cu[d]) : 0;
            const uint32_t has = __ballot_sync(0xffffffffu, (n + rows - 1) / rows > e);
            const int count = __popc(has);
            if (t < count) {
                *doc = d0 + __fns(has, 0, t + 1);
                *level = e;
                return true;
            }
            t -= count;
            found += count;
        }
        if (found == 0) return false;
    }
}

// tanh(scale s / cap) of a raw product s as 1 - 2 / (e^(2 s scale / cap) + 1).  The hardware's tanh is
// off by up to 2^-11, which a cap of 50 would turn into 3 % of a probability; this form is off by about 2e-7.
__device__ __forceinline__ float tanh_raw(const Attn& a, float s) {
    return fmaf(-2.0f, rcp_approx(ex2(s * a.tanh_in) + 1.0f), 1.0f);
}

// tanh(x) / x in x^2 on |x| <= 1/2: the polynomial of least largest relative error, 6.2e-7 in fp32 (iteratively reweighted
// least squares in the Chebyshev basis).
__device__ constexpr float kTanh[4] = {9.999994558e-01f, -3.332631793e-01f, 1.319029654e-01f, -4.440222454e-02f};
constexpr float kTanhEnd = 0.5f;

template <int N>
__device__ __forceinline__ float largest(const float (&s)[N]) {
    float a = fabsf(s[0]), b = fabsf(s[1]);
#pragma unroll
    for (int k = 2; k < N - 2; k += 4) {
        a = max3(a, fabsf(s[k]), fabsf(s[k + 1]));
        b = max3(b, fabsf(s[k + 2]), fabsf(s[k + 3]));
    }
    return max3(a, b, fmaxf(fabsf(s[N - 2]), fabsf(s[N - 1])));
}

// Raw products to tanh(scale s / cap).  Scores mostly stay well below their cap: where `fast` (no |scale s / cap| of the
// warp's above 1/2) a polynomial on the packed fp32 pipe takes 6 instructions a pair, against two trips through the
// special function unit an element.  The two differ in the last bits, so the choice must not follow from what a row does not
// see: columns with anything masked take the exact form, and rows behind the document have no say (capped, 8 x 1200 tokens,
// heads of 64: 126 -> 129 us; 2 x 2560 with prefix, heads of 128: 115 -> 119; masking the products before their largest is
// taken instead costs registers, and 140 and 120).
template <int N>
__device__ __forceinline__ void tanh_scores(const Attn& a, float (&s)[N], bool fast) {
    if (fast) {
        const uint64_t in2 = pack2(a.cap_in, a.cap_in);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const uint64_t x = mul2(pack2(s[k], s[k + 1]), in2), u = mul2(x, x);
            uint64_t p = pack2(kTanh[3], kTanh[3]);
#pragma unroll
            for (int i = 2; i >= 0; --i) p = fma2(p, u, pack2(kTanh[i], kTanh[i]));
            const float2 f = unpack2(mul2(p, x));
            s[k] = f.x;
            s[k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] = tanh_raw(a, s[k]);
    }
}
__device__ __forceinline__ bool tanh_fast(const Attn& a, float big) {
    return __all_sync(0xffffffffu, big * a.cap_in <= kTanhEnd);      // false for NaN
}

// s[k] c - slope |far - k|.  Where no row of the warp has its own place among the columns, the distance is linear in k.
template <int N>
__device__ __forceinline__ void bias_scores(float (&s)[N], float c, float slope, float far) {
    const bool behind = __all_sync(0xffffffffu, far >= (float)(N - 1)), ahead = __all_sync(0xffffffffu, far <= 0.0f);
    if (behind || ahead) {
        const float t = behind ? slope : -slope;              // s c - t far + t k
        const uint64_t c2 = pack2(c, c), t2 = pack2(t, t), b2 = pack2(-t * far, -t * far);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float2 f = unpack2(fma2(pack2(s[k], s[k + 1]), c2, fma2(t2, pack2((float)k, (float)(k + 1)), b2)));
            s[k] = f.x;
            s[k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] = fmaf(-slope, fabsf(far - (float)k), s[k] * c);
    }
}

// 2^x of a pair: the special function unit (16 a cycle and SM), or a polynomial on the fp32 pipe beside it.  2^x = 2^n 2^f,
// n the nearest integer (by adding 1.5 2^23, which leaves it in the low bits), f in [-1/2, 1/2]; 2^f = 1 + f q(f), q of
// degree 3 with least largest relative error of the whole, 2.9e-6 in fp32 (iteratively reweighted least squares in the
// Chebyshev basis); the factor 2^n is put together from its exponent field and multiplied, which keeps a NaN (adding n to
// the exponent field of 2^f does not).  x below -126.5, -inf with it, gives exactly 0 (n is -127 there, and the field 0);
// x up to 127; +inf and NaN give NaN.
__device__ __forceinline__ uint64_t ex2_poly(uint64_t x) {
    const float2 v = unpack2(x);
    x = pack2(max_nan(v.x, -127.0f), max_nan(v.y, -127.0f));
    const uint64_t t = add2(x, pack2(12582912.0f, 12582912.0f));
    const uint64_t f = fma2(add2(t, pack2(-12582912.0f, -12582912.0f)), pack2(-1.0f, -1.0f), x);
    uint64_t p = pack2(9.582852812e-03f, 9.582852812e-03f);
    p = fma2(p, f, pack2(5.590642500e-02f, 5.590642500e-02f));
    p = fma2(p, f, pack2(2.402409862e-01f, 2.402409862e-01f));
    p = fma2(p, f, pack2(6.931241933e-01f, 6.931241933e-01f));
    p = fma2(p, f, pack2(1.0f, 1.0f));
    const float2 tf = unpack2(t);
    return mul2(p, pack2(__int_as_float((__float_as_int(tf.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(tf.y) << 23) + 0x3f800000)));
}
// Which of 16 pairs take the polynomial: with `share` of them the fp32 pipe (2 cycles a packed instruction) and the special
// function unit (16 a pair) finish together.  A cap leaves the fp32 pipe no room.
__device__ __forceinline__ constexpr bool takes_poly(int k, int share) { return (k * share) % 16 < share; }

// Claims a block of this grid that has not started yet (its index becomes this CTA's next work); the 16-byte answer lands
// in `slot` and completes `bar`.
__device__ __forceinline__ void claim_block(uint64_t* slot, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(slot)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// The claimed block's x index, -1 where none was left.
__device__ __forceinline__ int claimed_block(const uint64_t* slot) {
    uint32_t x, got;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %1, 1, 0, p;\n\tmov.u32 %0, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
        : "=r"(x), "=r"(got)
        : "r"(smem_u32(slot))
        : "memory");
    return got ? (int)x : -1;
}

}  // namespace tok

// Host: fills an Attn and checks what every attention entry point checks.
int fill_attn(tok::Attn* a, int dtype, const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_len, int docs, int64_t Tq,
              int64_t Tk, int Hq, int Hk, int D, float scale, int causal, const int32_t* prefix, float softcap,
              const float* slopes, int32_t* status);

// Host: tensor map of [T, H, D] with a box of `rows` tokens of one head and 64 values.
int head_map(CUtensorMap* m, const void* p, int64_t tok, int64_t head, int64_t T, int H, int D, int rows);

}  // namespace pmg
