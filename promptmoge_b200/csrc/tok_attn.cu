// Attention over packed documents, forwards: rows by the tile (k_attn) and few rows over a long cache (k_attn_few).
//
// k_attn.  A CTA owns 256 query rows of one document and head, two tiles of 128 that share every key tile.  Products run on
// tcgen05 with the scores, the probabilities (left operand of the second product) and the running output in tensor memory;
// a thread has a row, so the softmax needs no shuffle.  The running maximum is only renewed, and the output only rescaled,
// when it has grown by more than 2^8: the probabilities then lie within 2^8, and the sums lose nothing to it.  Probabilities
// are rounded to the operands' 16-bit type for the second product (its operand can be no wider); the sums are of the
// unrounded ones, in fp32.  CTAs stay and claim the blocks of the grid that have not started: the next item's queries and
// keys are on their way while this one's output is stored.
//
// What bounds it is neither the tensor core (30 % active for heads of 64) nor the special function unit (46 %) but the chain
// of a step, scores -> maximum -> exponentials -> product -> next scores, with as many of them side by side as tensor memory
// and registers hold.  Measured: 16 frames of up to 1200 tokens, 16 heads of 64, fp16: 94 us (530 TFLOP/s); 16,384 tokens,
// 9 heads: 690 (warm) to 830 TFLOP/s with heads of 64, 1190 to 1200 with heads of 128.
#include <algorithm>
#include <cmath>

#include "tok_attn.cuh"

namespace pmg {

constexpr int64_t kMostTokens = INT32_MAX - 512;   // of a tensor: a tile's rows behind the last still have an int32 place

int fill_attn(tok::Attn* a, int dtype, const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_len, int docs, int64_t Tq,
              int64_t Tk, int Hq, int Hk, int D, float scale, int causal, const int32_t* prefix, float softcap,
              const float* slopes, int32_t* status) {
    if (dtype != PMG_F16 && dtype != PMG_BF16) return PMG_ERR_UNSUPPORTED;
    if (docs < 0 || Tq < 0 || Tk < 0 || Hq < 1 || Hk < 1 || Hq % Hk || D < 8 || !cu_q || !cu_k) return PMG_ERR_BAD_ARG;
    if (!(scale > 0.0f) || !std::isfinite(scale) || !(softcap >= 0.0f) || !std::isfinite(softcap)) return PMG_ERR_BAD_ARG;
    if (D % 8 || D > 128 || Tq > kMostTokens || Tk > kMostTokens || Hq > 65535) return PMG_ERR_UNSUPPORTED;
    *a = tok::Attn{};
    a->cu_q = cu_q; a->cu_k = cu_k; a->k_len = k_len; a->prefix = causal ? prefix : nullptr; a->slopes = slopes;
    a->Tq = Tq; a->Tk = Tk; a->docs = docs; a->Hq = Hq; a->Hk = Hk; a->group = Hq / Hk; a->D = D; a->causal = causal != 0;
    a->scale2 = scale * tok::kLog2e;
    a->cap2 = softcap * tok::kLog2e;
    a->tanh_in = softcap > 0.0f ? 2.0f * scale * tok::kLog2e / softcap : 0.0f;
    a->cap_in = softcap > 0.0f ? scale / softcap : 0.0f;
    a->status = status;
    return PMG_OK;
}

int head_map(CUtensorMap* m, const void* p, int64_t tok, int64_t head, int64_t T, int H, int D, int rows) {
    if ((tok & 7) || (head & 7)) return PMG_ERR_BAD_ARG;
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)H, (uint64_t)T};
    const uint64_t strides[2] = {(uint64_t)head * 2, (uint64_t)tok * 2};
    const uint32_t box[3] = {64, 1, (uint32_t)rows};
    return make_tensor_map16(m, p, 3, dims, strides, box);
}

namespace {

using namespace tok;

constexpr float kGrow = 8.0f;                  // log2 of how far scores may outgrow the running maximum

template <typename T> constexpr float kLift = 0.0f;
template <> constexpr float kLift<__half> = 7.0f;   // fp16 probabilities are kept times 2^7: 2^15 at most, and 7 more
                                                    // binades before they turn subnormal

template <typename T> constexpr float kUnlift = 1.0f;
template <> constexpr float kUnlift<__half> = 0.0078125f;

// A softmax thread has 64 columns of a row: what 96 registers hold, so that 16 softmax warps fit a SM, whose waits hide one
// another.  Heads up to 64: key tiles of 64, one warpgroup a row tile, two CTAs a SM (tensor memory: 2 (64 + 64) = 256 columns
// each), four row tiles at different points of their way.  Wider heads leave tensor memory for one CTA: key tiles of 128,
// two warpgroups a row tile, 2 (128 + 128) = 512 columns.
template <int DP>
struct Fwd {
    static constexpr int kHalves = DP == 64 ? 1 : 2;
    static constexpr int kCtas = DP == 64 ? 2 : 1;
    static constexpr int kBT = 64 * kHalves;                    // keys of a tile
    static constexpr int kThreads = 256 * kHalves + 64;         // softmax, then the loader and the MMA issuer
    static constexpr int kLoader = 8 * kHalves, kIssuer = kLoader + 1;
    static constexpr int kQTile = 128 * DP * 2, kQ = 2 * kQTile;
    static constexpr int kStrip = kBT * 128, kTile = kStrip * (DP / 64);
    static constexpr int kStages = DP == 64 ? 4 : 2;
    static constexpr int kBars = kQ + 2 * kStages * kTile;
    static constexpr int kTops = kBars + 1024; // what the two warpgroups of a row tile tell each other: [2][2][2][128]
    static constexpr int kSmem = kTops + (kHalves == 2 ? 4096 : 0);
    static constexpr uint32_t kCols = DP == 64 ? 256 : 512;
    static constexpr uint32_t S(int w) { return kBT * w; }
    static constexpr uint32_t P(int w, int h) { return kBT * w + 64 * h + 32; }   // over its own columns, from the end
    static constexpr uint32_t O(int w) { return 2 * kBT + DP * w; }
};

constexpr int kItems = 4;                      // items described ahead

// One item of a CTA's walk: 256 query rows of a document and head.
struct Item {
    int doc, head, r0, n0, n1;                 // doc < 0: the walk ends; n: key tiles of each half
    Span sp;
};

template <typename T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(Fwd<DP>::kThreads, Fwd<DP>::kCtas)
    k_attn(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
           const __grid_constant__ CUtensorMap mv, const __grid_constant__ Attn a, const int max_q, T* __restrict__ o,
           int64_t o_tok, int64_t o_head, float* __restrict__ lse) {
    using C = Fwd<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* const sk = smem + C::kQ;
    uint8_t* const sv = sk + C::kStages * C::kTile;
    uint64_t* const next_slot = reinterpret_cast<uint64_t*>(smem + C::kBars);      // 16 bytes: the answer to a claim
    uint64_t* const next_bar = next_slot + 2;
    uint64_t* const q_full = next_bar + 1;
    uint64_t* const q_empty = q_full + 2;
    uint64_t* const k_full = q_empty + 2;
    uint64_t* const k_empty = k_full + C::kStages;
    uint64_t* const v_full = k_empty + C::kStages;
    uint64_t* const v_empty = v_full + C::kStages;
    uint64_t* const s_full = v_empty + C::kStages;
    uint64_t* const p_full = s_full + 2;
    uint64_t* const pv_done = p_full + 2;
    uint64_t* const o_read = pv_done + 2;
    uint64_t* const told = o_read + 2;
    uint64_t* const item_full = told + 2;
    uint64_t* const item_empty = item_full + kItems;
    uint64_t* const drain = item_empty + kItems;
    Item* const items = reinterpret_cast<Item*>(drain + 1);
    uint32_t* const slot = reinterpret_cast<uint32_t*>(items + kItems);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 128 * C::kHalves);
            mbar_init(pv_done + i, 1);
            mbar_init(o_read + i, 128 * C::kHalves);
            mbar_init(told + i, 256);
        }
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(item_full + i, 1);
            mbar_init(item_empty + i, 8 * C::kHalves + 1);           // the softmax warps and the issuer
        }
        mbar_init(next_bar, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == C::kIssuer) tmem_alloc(slot, C::kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *slot, 0);
    pdl_begin();

    // Every warp but the loader reads the items in order through this.
    auto next_item = [&](uint32_t it, Item& x) -> bool {
        const int at = it % kItems;
        if (!__all_sync(0xffffffffu, wait_bar(item_full + at, (it / kItems) & 1u, abort_flag))) return false;
        x = items[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty + at);
        return true;
    };

    if (warp >= C::kLoader) {
        if (warp == C::kLoader) {
            // ------------------------------------------------------------------------------------------------ loads
            bool ok = true;
            uint32_t it = 0, kt = 0, qc[2] = {0, 0};
            int block = blockIdx.x;
            for (uint32_t claim = 0; block >= 0 && ok; ++claim) {
                if (lane == 0) claim_block(next_slot, next_bar);          // answered while this block is loaded
                Item x;
                x.doc = -1;
                int tile = 0;
                const bool found = a.causal ? find_level(a.cu_q, a.docs, 256, block / a.Hq, &x.doc, &tile)
                                            : find_tile(a.cu_q, a.docs, 256, block / a.Hq, &x.doc, &tile);
                if (found) {
                    x.sp = span_of(a, x.doc);
                    x.head = block % a.Hq;
                    // later rows of a causal document reach further: they start first
                    x.r0 = 256 * (a.causal ? (x.sp.lq + 255) / 256 - 1 - tile : tile);
                    if (x.r0 < 0) x.r0 = 1 << 30;                     // offsets that had to be cut: no such rows
                    x.n0 = x.r0 < x.sp.lq ? (key_end(a, x.sp, x.r0 + 128) + C::kBT - 1) / C::kBT : 0;
                    x.n1 = x.r0 + 128 < x.sp.lq ? (key_end(a, x.sp, x.r0 + 256) + C::kBT - 1) / C::kBT : 0;
                    const int at = it % kItems;
                    ok = __all_sync(0xffffffffu, wait_bar(item_empty + at, ((it / kItems) & 1u) ^ 1u, abort_flag));
                    if (!ok) break;
                    if (lane == 0) {
                        items[at] = x;
                        mbar_arrive(item_full + at);
                        const int kvh = x.head / a.group, nmax = max(x.n0, x.n1);
                        for (int w = 0; w < 2 && ok; ++w) {
                            if ((w ? x.n1 : x.n0) == 0) continue;
                            ok = wait_bar(q_empty + w, (qc[w] & 1u) ^ 1u, abort_flag);
                            if (!ok) break;
                            mbar_arrive_expect_tx(q_full + w, C::kQTile);
#pragma unroll
                            for (int c = 0; c < DP / 64; ++c)
                                tma_tile3d(smem_u32(smem + w * C::kQTile + c * 16384), &mq, 64 * c, x.head, x.sp.q0 + x.r0 + 128 * w, q_full + w);
                            ++qc[w];
                        }
                        for (int j = 0; j < nmax && ok; ++j, ++kt) {
                            const int st = kt % C::kStages;
                            const uint32_t ph = ((kt / C::kStages) & 1u) ^ 1u;
                            ok = wait_bar(k_empty + st, ph, abort_flag);
                            if (!ok) break;
                            mbar_arrive_expect_tx(k_full + st, C::kTile);
#pragma unroll
                            for (int c = 0; c < DP / 64; ++c)
                                tma_tile3d(smem_u32(sk + st * C::kTile + c * C::kStrip), &mk, 64 * c, kvh, x.sp.k0 + C::kBT * j, k_full + st);
                            ok = wait_bar(v_empty + st, ph, abort_flag);
                            if (!ok) break;
                            mbar_arrive_expect_tx(v_full + st, C::kTile);
#pragma unroll
                            for (int c = 0; c < DP / 64; ++c)
                                tma_tile3d(smem_u32(sv + st * C::kTile + c * C::kStrip), &mv, 64 * c, kvh, x.sp.k0 + C::kBT * j, v_full + st);
                        }
                    }
                    ++it;
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0);
                    if (!ok) break;
                }
                // there are as many blocks as documents, and more: each answers for one, which may have no tile at all
                if (block < a.docs) report_span(a, block, max_q);
                ok = __all_sync(0xffffffffu, wait_bar(next_bar, claim & 1u, abort_flag));
                if (!ok) break;
                block = claimed_block(next_slot);
                __syncwarp();
                fence_proxy_async();
            }
            if (ok) {
                const int at = it % kItems;
                ok = __all_sync(0xffffffffu, wait_bar(item_empty + at, ((it / kItems) & 1u) ^ 1u, abort_flag));
                if (ok && lane == 0) {
                    items[at].doc = -1;
                    mbar_arrive(item_full + at);
                }
            }
            if (!ok && lane == 0) {
                *abort_flag = 1;
                flag(a.status, PMG_ERR_TIMEOUT);
            }
        } else {
            // ------------------------------------------------------------------------------------------------ MMAs
            const int ksteps = (a.D + 15) / 16;
            const uint32_t id_qk = idesc16(Elem<T>::kFmt, 128, C::kBT, false, false);
            const uint32_t id_pv = idesc16(Elem<T>::kFmt, 128, ksteps * 16, false, true);
            const uint32_t lead = elect_one();
            bool ok = true;
            uint32_t kt = 0, qc[2] = {0, 0}, sc[2] = {0, 0};    // key tiles; items and tiles of each half so far
            auto wait = [&](uint64_t* bar, uint32_t ph) { return (bool)__all_sync(0xffffffffu, wait_bar(bar, ph & 1u, abort_flag)); };
            Item x;
            for (uint32_t it = 0;; ++it) {
                ok = next_item(it, x);
                if (!ok || x.doc < 0) break;
                const int n[2] = {__shfl_sync(0xffffffffu, x.n0, 0), __shfl_sync(0xffffffffu, x.n1, 0)}, nmax = max(n[0], n[1]);
                auto qk = [&](int w, int j) -> bool {
                    const uint32_t t = kt + j, st = t % C::kStages;
                    if (j == 0 && !wait(q_full + w, qc[w])) return false;
                    if (!wait(k_full + st, t / C::kStages)) return false;
                    tc_fence_after();
                    const uint32_t qa = desc_lo(smem_u32(smem + w * C::kQTile), 16), kb = desc_lo(smem_u32(sk + st * C::kTile), 16);
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
                        if (s < ksteps) {
                            const uint32_t in = (s & 3) * 2;
                            mma16(lead, tmem + C::S(w), qa + (s >> 2) * 1024 + in, kb + (s >> 2) * (C::kStrip / 16) + in, id_qk, s > 0);
                        }
                    mma_commit_if(lead, s_full + w);
                    if (w == 1 || j >= n[1]) mma_commit_if(lead, k_empty + st);     // the tile's last reader
                    if (j + 1 == n[w]) mma_commit_if(lead, q_empty + w);
                    return true;
                };
                auto pv = [&](int w, int j) -> bool {
                    const uint32_t t = kt + j, st = t % C::kStages;
                    if (!wait(v_full + st, t / C::kStages)) return false;
                    const int valid = x.sp.lk - C::kBT * j;
                    if (valid < C::kBT && (w == 0 || n[0] <= j)) {
                        // rows behind the document's last key: whatever lies there must not reach a sum (0 * NaN)
                        for (int c = 0; c < DP / 64; ++c)
                            for (int b = valid * 128 + lane * 16; b < C::kStrip; b += 512)
                                *reinterpret_cast<uint4*>(sv + st * C::kTile + c * C::kStrip + b) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                    }
                    if (j == 0 && !wait(o_read + w, qc[w] ^ 1u)) return false;    // the last item's output is out
                    tc_fence_after();
                    const uint32_t vb = desc_lo(smem_u32(sv + st * C::kTile), C::kStrip);
#pragma unroll
                    for (int s = 0; s < C::kBT / 16; ++s)
                        mma16_ts(lead, tmem + C::O(w), tmem + C::P(w, s >> 2) + 8 * (s & 3), vb + s * 128, id_pv, j > 0 || s > 0);
                    mma_commit_if(lead, pv_done + w);
                    if (w == 1 || j >= n[1]) mma_commit_if(lead, v_empty + st);
                    return true;
                };
                for (int w = 0; w < 2 && ok; ++w)
                    if (n[w] > 0) ok = qk(w, 0);
                for (int j = 0; j < nmax && ok; ++j) {
                    // Each row tile on its own: its product and its next scores (over its probabilities) follow when its
                    // softmax is through, while the other's runs.
                    for (int w = 0; w < 2 && ok; ++w) {
                        if (j >= n[w]) continue;
                        ok = wait(p_full + w, sc[w] + j);
                        if (ok) ok = pv(w, j);
                        if (ok && j + 1 < n[w]) ok = qk(w, j + 1);
                    }
                }
                if (!ok) break;
                kt += nmax;
                for (int w = 0; w < 2; ++w) {
                    sc[w] += n[w];
                    qc[w] += n[w] > 0;
                }
            }
            if (lane == 0) {
                if (!ok) flag(a.status, PMG_ERR_TIMEOUT);
                if (!ok || *abort_flag) {
                    *abort_flag = 1;
                    drain_mma(drain);
                }
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------------------------------------- softmax
        // Where two warpgroups share a row tile they tell each other their maxima (and at the end their sums) through shared
        // memory, take the same maximum, and rescale and store half the output each.
        const int w = (warp >> 2) / C::kHalves, h = (warp >> 2) % C::kHalves;
        constexpr int kOut = DP / C::kHalves;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + C::S(w) + 64 * h, tp = tmem + lanes + C::P(w, h), to = tmem + lanes + C::O(w) + h * kOut;
        float* const tops = reinterpret_cast<float*>(smem + C::kTops) + w * 256 + (warp & 3) * 32 + lane;
        const float c = BIAS ? 1.0f : (CAP ? a.cap2 : a.scale2);          // scores to units of log 2
        uint32_t sc = 0, xc = 0;                                          // tiles; exchanges
        bool ok = true;
        auto tell = [&](float v) {
            tops[(xc & 1) * 512 + h * 128] = v;
            mbar_arrive(told + w);
        };
        auto hear = [&](float& v) {                                       // false: gave up
            if (!__all_sync(0xffffffffu, wait_bar(told + w, xc & 1u, abort_flag))) return false;
            v = tops[(xc & 1) * 512 + (h ^ 1) * 128];
            ++xc;
            return true;
        };
        Item x;
        for (uint32_t it = 0;; ++it) {
            ok = next_item(it, x);
            if (!ok || x.doc < 0) break;
            const int tiles_k = w ? x.n1 : x.n0;
            const int i = x.r0 + 128 * w + (warp & 3) * 32 + lane;        // this thread's row in the document
            const int lim = last_key(a, x.sp, i);
            const int warp_min = __reduce_min_sync(0xffffffffu, i < x.sp.lq ? lim : INT32_MAX);
            const float slope = BIAS ? a.slopes[x.head] * kLog2e : 0.0f;
            const float place = (float)(i + x.sp.lk - x.sp.lq);
            float m = -INFINITY;
            uint64_t sum = 0, sum2 = 0;
            for (int j = 0; j < tiles_k; ++j, ++sc) {
                TOK_WAIT(s_full + w, sc & 1u);
                if (!ok) break;
                tc_fence_after();
                const int j0 = C::kBT * j + 64 * h;
                // 32 columns at a time: the first are read again for their probabilities, which costs less than the
                // registers to keep them.
                float s[32];
                bool fast = false;                        // the cap's polynomial serves (tanh_fast)
                const bool masked = j0 + 63 > warp_min;   // something of these columns is hidden from a row of the warp
                auto fetch = [&](int q) {
                    tmem_ld32(ts + 32 * q, reinterpret_cast<uint32_t*>(s));
                    tmem_wait_ld();
                };
                auto mask = [&](int q) {
                    if (j0 + 32 * q + 31 > warp_min) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (j0 + 32 * q + k > lim) s[k] = -INFINITY;
                    }
                };
                auto score = [&](int q) {                 // raw products to what the softmax takes
                    if (CAP) tanh_scores<32>(a, s, BIAS ? j0 + 32 * q + 31 <= warp_min && tanh_fast(a, lim >= 0 ? largest<32>(s) : 0.0f) : fast);
                    if (BIAS) bias_scores<32>(s, CAP ? a.cap2 : a.scale2, slope, place - (float)(j0 + 32 * q));
                    mask(q);
                };
                float top = -INFINITY, top2 = -INFINITY, big = 0.0f;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    fetch(q);
                    if (CAP && !BIAS) big = fmaxf(big, largest<32>(s));
                    if (BIAS) score(q);
                    else mask(q);                         // a cap keeps the order: the maximum is capped afterwards
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        top = max3(top, s[k], s[k + 1]);
                        top2 = max3(top2, s[k + 2], s[k + 3]);
                    }
                }
                top = fmaxf(top, top2);
                if (C::kHalves == 2) tell(top);
                if (CAP && !BIAS) {
                    fast = !masked && tanh_fast(a, lim >= 0 ? big : 0.0f);
                    score(1);
                }
                if (C::kHalves == 2) {
                    float other = 0.0f;
                    ok = hear(other);
                    if (!ok) break;
                    top = fmaxf(top, other);
                }
                // where the row sees a key of this tile: a raw product of -inf stands for -cap, not for no key
                if (CAP && !BIAS && C::kBT * j <= lim) top = tanh_raw(a, top);
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, (top - m) * c > kGrow)) {
                    // only the rows that grew, so that no row's bits follow from what its neighbours see
                    if (!((top - m) * c > kGrow)) top = m;
                    const float f = top == m ? 1.0f : ex2((m - top) * c);
                    m = top;
                    sum = mul2(sum, pack2(f, f));
                    sum2 = mul2(sum2, pack2(f, f));
                    tc_fence_after();
#pragma unroll
                    for (int q = 0; q < kOut / 16; ++q) {
                        uint32_t v[16];
                        tmem_ld16(to + 16 * q, v);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                        tmem_st16(to + 16 * q, v);
                    }
                }
                const float base = m == -INFINITY ? 0.0f : -m * c + kLift<T>;
                const uint64_t c2 = pack2(c, c), b2 = pack2(base, base);
                auto exps = [&](int q) {
                    uint32_t p[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const uint64_t y = fma2(pack2(s[2 * k], s[2 * k + 1]), c2, b2);
                        const uint64_t e = takes_poly(k, CAP ? 0 : 4) ? ex2_poly(y) : ex2_pair(y);
                        if (k & 1) sum2 = add2(sum2, e);
                        else sum = add2(sum, e);
                        const float2 f = unpack2(e);
                        p[k] = Elem<T>::pack(f.x, f.y);
                    }
                    tmem_st16(tp + 16 * q, p);
                };
                exps(1);
                fetch(0);
                score(0);
                exps(0);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(p_full + w);
            }
            if (!ok) break;
            const float2 s2 = unpack2(add2(sum, sum2));
            float total = s2.x + s2.y, rest = 0.0f;
            if (C::kHalves == 2) {
                tell(total);
                ok = hear(rest);
                if (!ok) break;
                total = h ? rest + total : total + rest;
            }
            if (tiles_k > 0) TOK_WAIT(pv_done + w, (sc - 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            const int64_t token = x.sp.q0 + (int64_t)i;
            const bool mine = i < x.sp.lq, none = total == 0.0f;         // rows that see no key give zero
            const float inv = none ? 0.0f : 1.0f / total;
            if (mine && h == 0) lse[(int64_t)x.head * a.Tq + token] = none ? -INFINITY : (m * c + log2f(total * kUnlift<T>)) * kLn2;
            T* row = o + token * o_tok + x.head * o_head + h * kOut;
#pragma unroll
            for (int q = 0; q < kOut / 32; ++q) {
                float v[32];
                if (tiles_k > 0) {
                    tmem_ld32(to + 32 * q, reinterpret_cast<uint32_t*>(v));
                    tmem_wait_ld();
                }
                if (q == kOut / 32 - 1 && tiles_k > 0) {
                    tc_fence_before();
                    mbar_arrive(o_read + w);
                }
                if (none) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (mine && h * kOut + 32 * q + 8 * k < a.D)
                        *reinterpret_cast<uint4*>(row + 32 * q + 8 * k) =
                            make_uint4(Elem<T>::pack(v[8 * k] * inv, v[8 * k + 1] * inv),
                                       Elem<T>::pack(v[8 * k + 2] * inv, v[8 * k + 3] * inv),
                                       Elem<T>::pack(v[8 * k + 4] * inv, v[8 * k + 5] * inv),
                                       Elem<T>::pack(v[8 * k + 6] * inv, v[8 * k + 7] * inv));
            }
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            flag(a.status, PMG_ERR_TIMEOUT);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == C::kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kCols);
    }
}

// ----------------------------------------------------------------------------------------------------------------- //
// Few rows over many keys
// ----------------------------------------------------------------------------------------------------------------- //
// Bound by one read of the keys and values.  A CTA takes one document, one key head and a stretch of the keys; the up to
// 16 query rows that share the key head (queries x group) are the 16 rows of mma.sync, so every key is read once for all
// of them.  One warp keeps a ring of 64-key tiles filled by TMA, 64 to 96 KB of them in flight a CTA and two or three CTAs
// a SM; four warps take 16 keys of each tile, on their own, through ldmatrix (TMA's 128-byte swizzle is the one that
// makes it free of bank conflicts).  Loading straight into registers, with the wait for each block's loads in the open,
// read 1.7 TB/s; this reads 4.8 TB/s (32 streams over up to 8192 tokens, 4 key heads of 64) and 5.0 TB/s (65,501 keys, 4 key
// heads of 128).  Warps, then stretches, are joined by their maxima and sums.

constexpr int kFewWarps = 4, kFewRows = 16, kFewTile = 64, kFewThreads = 32 * (kFewWarps + 1);

template <int DP>
struct Few {
    static constexpr int kPart = kFewTile * DP * 2;               // a tile's keys, or values
    static constexpr int kStages = DP == 64 ? 4 : 3;
    static constexpr int kBars = kStages * 2 * kPart;
    static constexpr int kSmem = kBars + 256;
    static constexpr int kCtas = DP == 64 ? 3 : 2;                // a SM
};

template <typename T>
__device__ __forceinline__ void mma_16n8k16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (Elem<T>::kFmt == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

struct Heads {                    // [T, H, D]: pointer and strides in elements
    const void* p;
    int64_t tok, head;
};

// Partial results of a stretch: per row D unnormalised outputs, then maximum and sum (units of log 2).
template <typename T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kFewThreads, Few<DP>::kCtas)
    k_attn_few(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Heads hq,
               const __grid_constant__ Attn a, int max_q, int stretch, float* __restrict__ part, T* __restrict__ o,
               int64_t o_tok, int64_t o_head, float* __restrict__ lse) {
    using C = Few<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* const full = reinterpret_cast<uint64_t*>(smem + C::kBars);
    uint64_t* const empty = full + C::kStages;
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(empty + C::kStages);
    const int split = blockIdx.x, splits = gridDim.x, kvh = blockIdx.y, doc = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kFewWarps);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    pdl_begin();
    bool bad;
    const Span sp = cut_span(a, doc, &bad);
    if ((bad || sp.lq > max_q) && threadIdx.x == 0) flag(a.status, PMG_ERR_RANGE);
    const int rows = min(sp.lq, max_q) * a.group;
    const int reach = key_end(a, sp, sp.lq), kbeg = split * stretch;
    const int kend = split + 1 < splits ? min(reach, kbeg + stretch) : reach;       // the last takes what max_k left out
    if (rows == 0 || (kbeg >= reach && split > 0)) return;            // the first stretch also stands for no keys at all
    const int tiles = kend > kbeg ? (kend - kbeg + kFewTile - 1) / kFewTile : 0;
    __syncthreads();

    float acc[DP / 8][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const float c = BIAS ? 1.0f : (CAP ? a.cap2 : a.scale2);
    bool ok = true;
    if (warp == kFewWarps) {
        if (lane == 0) {
            int i = 0;
            for (; i < tiles; ++i) {
                const int st = i % C::kStages;
                ok = mbar_wait(empty + st, ((i / C::kStages) & 1u) ^ 1u, abort_flag);
                if (!ok) break;
                const uint32_t to = smem_u32(smem + st * 2 * C::kPart);
                mbar_arrive_expect_tx(full + st, 2 * C::kPart);
#pragma unroll
                for (int x = 0; x < DP / 64; ++x) {
                    tma_tile3d(to + x * 8192, &mk, 64 * x, kvh, sp.k0 + kbeg + kFewTile * i, full + st);
                    tma_tile3d(to + C::kPart + x * 8192, &mv, 64 * x, kvh, sp.k0 + kbeg + kFewTile * i, full + st);
                }
            }
            // all has landed before the ring's room takes the warps' rows, or the block leaves, also after an abort
            const uint64_t t0 = global_ns();
            for (int n = max(i - C::kStages, 0); n < i; ++n)
                while (!mbar_try_wait_sleep(full + n % C::kStages, (n / C::kStages) & 1u, 4000) && global_ns() - t0 < kWaitNs) {
                }
        }
    } else {
        // queries: rows g and g + 8 as left operands
        uint32_t qf[DP / 16][4];
        int lim[2], whole = INT32_MAX;                   // whole: the last key that every row sees
        float place[2], slope[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h, i = r / a.group, hd = kvh * a.group + r % a.group;
            const bool on = r < rows;
            lim[h] = on ? min(last_key(a, sp, i), kend - 1) : -1;
            if (on) whole = min(whole, lim[h]);
            place[h] = (float)(i + sp.lk - sp.lq);
            slope[h] = BIAS && on ? a.slopes[hd] * kLog2e : 0.0f;
            const T* p = static_cast<const T*>(hq.p) + (sp.q0 + (int64_t)i) * hq.tok + hd * hq.head;
#pragma unroll
            for (int x = 0; x < DP / 16; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 16 * x + 8 * e + 2 * q;
                    qf[x][h + 2 * e] = on && d < a.D ? *reinterpret_cast<const uint32_t*>(p + d) : 0u;
                }
        }
        whole = __reduce_min_sync(0xffffffffu, whole);
        // ldmatrix: lane l gives the row of matrix l / 8; K: (keys 0-7, 8-15) x (first, second 8 values), V: the same rows
        const int kr = warp * 16 + (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
        const int vr = warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
        for (int i = 0; i < tiles; ++i) {
            const int st = i % C::kStages, j0 = kbeg + kFewTile * i + 16 * warp;      // this warp's first key
            ok = __all_sync(0xffffffffu, mbar_wait(full + st, (i / C::kStages) & 1u, abort_flag));
            if (!ok) break;
            uint8_t* const kt = smem + st * 2 * C::kPart;
            uint8_t* const vt = kt + C::kPart;
            if (j0 < kend) {
                float s[8] = {};                         // row tile x 8 keys, as the instruction leaves them: 4 t + e
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    uint32_t b[4];
                    ldmatrix4<false>(b, smem_u32(kt) + (x >> 2) * 8192 + kr * 128 + ((((x & 3) * 2 + kc) ^ (kr & 7)) << 4));
                    mma_16n8k16<T>(*reinterpret_cast<float (*)[4]>(s), qf[x], b[0], b[1]);
                    mma_16n8k16<T>(*reinterpret_cast<float (*)[4]>(s + 4), qf[x], b[2], b[3]);
                }
                if (j0 + 16 > kend) {
                    // rows behind the last key: whatever lies there must not reach a sum (0 * NaN)
                    for (int x = lane; x < 16 * (DP / 8); x += 32) {
                        const int r = x & 15;
                        if (j0 + r >= kend)
                            *reinterpret_cast<uint4*>(vt + (x >> 7) * 8192 + (warp * 16 + r) * 128 + ((x >> 4) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                // as by the tile: keys hidden from a row have no part in the choice of tanh's form
                if (CAP) tanh_scores<8>(a, s, j0 + 15 <= whole && tanh_fast(a, largest<8>(s)));
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int h = e >> 1, key = j0 + 8 * t + 2 * q + (e & 1);
                        float x = s[4 * t + e];
                        if (BIAS) x = fmaf(-slope[h], fabsf(place[h] - (float)key), x * (CAP ? a.cap2 : a.scale2));
                        x = key <= lim[h] ? x : -INFINITY;
                        s[4 * t + e] = x;
                        top[h] = fmaxf(top[h], x);
                    }
                bool grew[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    grew[h] = (top[h] - m[h]) * c > kGrow;
                }
                if (__any_sync(0xffffffffu, grew[0] || grew[1])) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float f = grew[h] ? ex2((m[h] - top[h]) * c) : 1.0f;
                        if (grew[h]) m[h] = top[h];
                        l[h] *= f;
#pragma unroll
                        for (int x = 0; x < DP / 8; ++x) {
                            acc[x][2 * h] *= f;
                            acc[x][2 * h + 1] *= f;
                        }
                    }
                }
                uint32_t p[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float base = m[h] == -INFINITY ? 0.0f : -m[h] * c + kLift<T>;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float e0 = ex2(fmaf(s[4 * t + 2 * h], c, base)), e1 = ex2(fmaf(s[4 * t + 2 * h + 1], c, base));
                        l[h] += e0 + e1;
                        p[2 * t + h] = Elem<T>::pack(e0, e1);
                    }
                }
#pragma unroll
                for (int x = 0; x < DP / 16; ++x) {
                    uint32_t b[4];
                    ldmatrix4<true>(b, smem_u32(vt) + (x >> 2) * 8192 + vr * 128 + ((((x & 3) * 2 + vc) ^ (vr & 7)) << 4));
                    mma_16n8k16<T>(acc[2 * x], p, b[0], b[1]);
                    mma_16n8k16<T>(acc[2 * x + 1], p, b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + st);
        }
    }
    if (!ok && lane == 0) {
        *abort_flag = 1;
        flag(a.status, PMG_ERR_TIMEOUT);
    }
    __syncthreads();                                  // every tile has been read: its room takes the warps' rows
    float* const sm = reinterpret_cast<float*>(smem); // [warps][16][DP], then [warps][16] maxima, [warps][16] sums
    float* const sm_m = sm + kFewWarps * kFewRows * DP;
    float* const sm_l = sm_m + kFewWarps * kFewRows;
    if (warp < kFewWarps) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int r = warp * kFewRows + g + 8 * h;
            if (q == 0) {
                sm_m[r] = m[h] * c;
                sm_l[r] = l[h];
            }
#pragma unroll
            for (int x = 0; x < DP / 8; ++x)
                *reinterpret_cast<float2*>(sm + r * DP + 8 * x + 2 * q) = make_float2(acc[x][2 * h], acc[x][2 * h + 1]);
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows * (DP / 4); idx += blockDim.x) {
        const int r = idx / (DP / 4), d = (idx % (DP / 4)) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, sm_m[w * kFewRows + r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float total = 0.0f;
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float f = ex2(sm_m[w * kFewRows + r] - ref);
            const float4 x = *reinterpret_cast<const float4*>(sm + (w * kFewRows + r) * DP + d);
            total += f * sm_l[w * kFewRows + r];
            v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
        }
        if (splits > 1) {
            float* to = part + ((((int64_t)doc * a.Hk + kvh) * splits + split) * kFewRows + r) * (DP + 4);
            *reinterpret_cast<float4*>(to + d) = v;
            if (d == 0) {
                to[DP] = top;
                to[DP + 1] = total;
            }
            continue;
        }
        const int64_t token = sp.q0 + (int64_t)(r / a.group);
        const int head = kvh * a.group + r % a.group;
        if (d >= a.D) continue;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        *reinterpret_cast<uint2*>(o + token * o_tok + head * o_head + d) =
            make_uint2(Elem<T>::pack(v.x * inv, v.y * inv), Elem<T>::pack(v.z * inv, v.w * inv));
        if (d == 0) lse[(int64_t)head * a.Tq + token] = total == 0.0f ? -INFINITY : (top + log2f(total * kUnlift<T>)) * kLn2;
    }
}

// Joins the stretches of a row, a block a row: a strand of DP / 4 threads takes every 256 / (DP / 4)-th stretch, the
// strands are added in order.  (A warp a row walked 74 stretches in 28 us, as long as the keys themselves took.)
template <typename T, int DP>
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ Attn a, int max_q, int room, int stretch,
                                                   const float* __restrict__ part, T* __restrict__ o, int64_t o_tok,
                                                   int64_t o_head, float* __restrict__ lse) {
    pdl_begin();
    constexpr int kWide = DP / 4, kStrands = 256 / kWide;
    __shared__ float sm_top[8], sm_sum[kStrands];
    __shared__ float4 sm[kStrands][kWide];
    const int r = blockIdx.x, kvh = blockIdx.y, doc = blockIdx.z, x = threadIdx.x % kWide, strand = threadIdx.x / kWide;
    const Span sp = span_of(a, doc);
    if (r >= min(sp.lq, max_q) * a.group) return;
    const int splits = min(room, max(1, (key_end(a, sp, sp.lq) + stretch - 1) / stretch));
    const float* from = part + (((int64_t)doc * a.Hk + kvh) * room * kFewRows + r) * (DP + 4);
    constexpr int64_t step = kFewRows * (DP + 4);
    float top = -INFINITY;
    for (int s = threadIdx.x; s < splits; s += 256) top = fmaxf(top, from[s * step + DP]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    if ((threadIdx.x & 31) == 0) sm_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, sm_top[k]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int s = strand; s < splits; s += kStrands) {
        const float f = ex2(from[s * step + DP] - ref);
        const float4 y = *reinterpret_cast<const float4*>(from + s * step + 4 * x);
        total += f * from[s * step + DP + 1];
        v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
    }
    sm[strand][x] = v;
    if (x == 0) sm_sum[strand] = total;
    __syncthreads();
    if (strand) return;
    total = 0.0f;
    v = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kStrands; ++k) {
        const float4 y = sm[k][x];
        total += sm_sum[k];
        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    const int64_t token = sp.q0 + (int64_t)(r / a.group);
    const int head = kvh * a.group + r % a.group, d = 4 * x;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if (d < a.D)
        *reinterpret_cast<uint2*>(o + token * o_tok + head * o_head + d) =
            make_uint2(Elem<T>::pack(v.x * inv, v.y * inv), Elem<T>::pack(v.z * inv, v.w * inv));
    if (x == 0) lse[(int64_t)head * a.Tq + token] = total == 0.0f ? -INFINITY : (top + log2f(total * kUnlift<T>)) * kLn2;
}

// ----------------------------------------------------------------------------------------------------------------- //
// Host side
// ----------------------------------------------------------------------------------------------------------------- //
template <auto KERNEL>
int raise_smem(int bytes) {
    static bool set[64] = {};
    int dev = 0;
    PMG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return PMG_ERR_UNSUPPORTED;
    if (!set[dev]) {
        PMG_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        set[dev] = true;
    }
    return PMG_OK;
}

struct Call {
    Heads q, k, v;
    void* o;
    int64_t o_tok, o_head;
    float* lse;
    int max_q, max_k;
    float* part;
};

bool few_rows(int max_q, int group) { return (int64_t)max_q * group <= kFewRows; }

// Keys of a stretch, a multiple of a tile: one round of the CTAs that fit the GPU together for one document, a quarter of
// that for several, whose lengths differ (CTAs then take turns and even out); at least 256, so that a stretch is longer
// than its start, and no more than all of them.  No document holds more keys than a tensor may; a larger bound counts as that.
int few_stretch(int docs, int Hk, int D, int max_k) {
    const int64_t most = std::min<int64_t>(max_k, kMostTokens);
    const int64_t slots = (int64_t)kNumSMs * (D <= 64 ? Few<64>::kCtas : Few<128>::kCtas) * (docs > 1 ? 4 : 1);
    const int64_t pairs = (int64_t)docs * Hk, keys = pairs >= slots ? most : (pairs * most + slots - 1) / slots;
    return (int)((std::max<int64_t>(keys, 256) + kFewTile - 1) / kFewTile * kFewTile);
}
int few_splits(int docs, int Hk, int D, int max_k) {
    const int64_t most = std::min<int64_t>(max_k, kMostTokens), stretch = few_stretch(docs, Hk, D, max_k);
    return (int)std::max<int64_t>(1, (most + stretch - 1) / stretch);
}

template <typename T, int DP, bool CAP, bool BIAS>
int run(const Attn& a, const Call& c, cudaStream_t s) {
    if (few_rows(c.max_q, a.group)) {
        const int stretch = few_stretch(a.docs, a.Hk, a.D, c.max_k), splits = few_splits(a.docs, a.Hk, a.D, c.max_k);
        const int rc = raise_smem<k_attn_few<T, DP, CAP, BIAS>>(Few<DP>::kSmem);
        if (rc != PMG_OK) return rc;
        CUtensorMap mk, mv;
        int e = head_map(&mk, c.k.p, c.k.tok, c.k.head, std::max<int64_t>(a.Tk, 1), a.Hk, a.D, kFewTile);
        if (e == PMG_OK) e = head_map(&mv, c.v.p, c.v.tok, c.v.head, std::max<int64_t>(a.Tk, 1), a.Hk, a.D, kFewTile);
        if (e != PMG_OK) return e;
        for (int d0 = 0; d0 < a.docs; d0 += 65535) {
            Attn b = a;
            b.docs = std::min(65535, a.docs - d0);
            b.cu_q += d0;
            b.cu_k += d0;
            if (b.k_len) b.k_len += d0;
            if (b.prefix) b.prefix += d0;
            k_attn_few<T, DP, CAP, BIAS><<<dim3(splits, a.Hk, b.docs), kFewThreads, Few<DP>::kSmem, s>>>(
                mk, mv, c.q, b, c.max_q, stretch, c.part, static_cast<T*>(c.o), c.o_tok, c.o_head, c.lse);
            PMG_LAUNCH_CHECK();
            if (splits > 1) {
                const int rc2 = launch_after(k_attn_join<T, DP>, dim3(c.max_q * a.group, a.Hk, b.docs), 256, 0, s, b, c.max_q,
                                             splits, stretch, (const float*)c.part, static_cast<T*>(c.o), c.o_tok, c.o_head, c.lse);
                if (rc2 != PMG_OK) return rc2;
            }
        }
        return PMG_OK;
    }
    using C = Fwd<DP>;
    const int rc = raise_smem<k_attn<T, DP, CAP, BIAS>>(C::kSmem);
    if (rc != PMG_OK) return rc;
    CUtensorMap mq, mk, mv;
    int e = head_map(&mq, c.q.p, c.q.tok, c.q.head, a.Tq, a.Hq, a.D, 128);
    if (e == PMG_OK) e = head_map(&mk, c.k.p, c.k.tok, c.k.head, std::max<int64_t>(a.Tk, 1), a.Hk, a.D, C::kBT);
    if (e == PMG_OK) e = head_map(&mv, c.v.p, c.v.tok, c.v.head, std::max<int64_t>(a.Tk, 1), a.Hk, a.D, C::kBT);
    if (e != PMG_OK) return e;
    const int64_t blocks = (a.Tq / 256 + a.docs) * a.Hq;
    if (blocks > INT32_MAX) return PMG_ERR_UNSUPPORTED;
    k_attn<T, DP, CAP, BIAS><<<(int)blocks, C::kThreads, C::kSmem, s>>>(mq, mk, mv, a, c.max_q, static_cast<T*>(c.o), c.o_tok, c.o_head, c.lse);
    PMG_LAUNCH_CHECK();
    return PMG_OK;
}

template <typename T, int DP>
int by_score(const Attn& a, const Call& c, cudaStream_t s) {
    if (a.cap2 > 0.0f) return a.slopes ? run<T, DP, true, true>(a, c, s) : run<T, DP, true, false>(a, c, s);
    return a.slopes ? run<T, DP, false, true>(a, c, s) : run<T, DP, false, false>(a, c, s);
}

}  // namespace
}  // namespace pmg

using namespace pmg;

extern "C" size_t pmg_attention_workspace_bytes(int32_t docs, int32_t Hq, int32_t Hk, int32_t D, int32_t max_q,
                                                int32_t max_k) {
    if (docs < 1 || Hk < 1 || Hq < Hk || max_q < 1 || !few_rows(max_q, Hq / Hk)) return 0;
    const int splits = few_splits(docs, Hk, D, max_k);
    return splits > 1 ? (size_t)std::min(docs, 65535) * Hk * splits * kFewRows * ((D <= 64 ? 64 : 128) + 4) * sizeof(float) : 0;
}

extern "C" int pmg_attention(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok,
                             int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, int32_t dtype, int64_t Tq,
                             int64_t Tk, int32_t Hq, int32_t Hk, int32_t D, const int32_t* cu_q, const int32_t* cu_k,
                             const int32_t* k_len, int32_t docs, int32_t max_q, int32_t max_k, float scale,
                             int32_t causal, const int32_t* prefix, float softcap, const float* slopes, void* o,
                             int64_t o_tok, int64_t o_head, float* lse, void* workspace, size_t workspace_bytes,
                             int32_t* status, void* stream) {
    Attn a;
    const int rc = fill_attn(&a, dtype, cu_q, cu_k, k_len, docs, Tq, Tk, Hq, Hk, D, scale, causal, prefix, softcap, slopes, status);
    if (rc != PMG_OK) return rc;
    if (docs == 0 || Tq == 0) return PMG_OK;
    if (Tk == 0) {                    // nothing is read of the keys: any valid place serves their tensor maps
        k = v = q;
        k_tok = v_tok = q_tok;
        k_head = v_head = q_head;
    }
    if (!q || !k || !v || !o || !lse || max_q < 0 || max_k < 0) return PMG_ERR_BAD_ARG;
    auto ok = [](const void* p, int64_t t, int64_t h) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(t & 7) && !(h & 7); };
    if (!ok(q, q_tok, q_head) || !ok(k, k_tok, k_head) || !ok(v, v_tok, v_head) || !ok(o, o_tok, o_head)) return PMG_ERR_BAD_ARG;
    if (max_q == 0) max_k = 0;        // one short launch a document, which reports those that do have queries
    const size_t need = pmg_attention_workspace_bytes(docs, Hq, Hk, D, max_q, max_k);
    if (workspace_bytes < need || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))) return PMG_ERR_BAD_ARG;
    Call c{{q, q_tok, q_head}, {k, k_tok, k_head}, {v, v_tok, v_head}, o, o_tok, o_head, lse, max_q, max_k, static_cast<float*>(workspace)};
    cudaStream_t s = as_stream(stream);
    if (dtype == PMG_BF16) return D <= 64 ? by_score<__nv_bfloat16, 64>(a, c, s) : by_score<__nv_bfloat16, 128>(a, c, s);
    return D <= 64 ? by_score<__half, 64>(a, c, s) : by_score<__half, 128>(a, c, s);
}
