// Gradients of attention over packed documents.
//
//   P = exp(s - lse), dV = P^T dO, dP = dO V^T, dS = P (dP - delta), delta = rowsum(dO o),
//   through the cap: dS (1 - (s_c / cap)^2);  dQ = scale dS K, dK = scale dS^T Q, the shared key heads' sums over their
//   group taken by the kernel that owns the keys.
//
// One launch, two kinds of CTA, each with 128 stationary rows: keys (dK, dV; streams the queries of all heads that share
// the key head) and queries (dQ; streams the keys).  Both compute scores and dP with their own rows in tensor-memory
// lanes, so the probabilities and dS are left operands where they stand, in the columns their inputs leave, and nothing
// is transposed or sent through shared memory.  Scores are computed twice for it (7 products a tile instead of 5), and
// in return no gradient is summed by atomics: results do not depend on timing, and no fp32 copy of dQ is kept.
// P and dS are rounded to the operands' 16-bit type (tensor cores take no other); fp16 values are kept times a power of
// two, 2^15 for P (which is at most 1) and for dS the one that |dS| <= 2 max|dO| max|V| over its document allows, so that
// small gradients do not turn subnormal.
//
// Bound by the chain of a step, as forwards (tensor core 37 % active, issue slots 59 %).  Measured: 8 frames of up to 1200
// tokens, 16 heads of 64 over 4 key heads, distance bias: 175 us; 8192 tokens, 16 heads of 64: 715 (warm) to 750
// TFLOP/s of the 5 products that the gradient needs, heads of 128: 815 to 870.
#include <algorithm>

#include "tok_attn.cuh"

namespace pmg {
namespace {

using namespace tok;

// The factor that fp16 dS carries follows from a document's largest |dO| and |V|, of its own rows alone, so that neither
// another document nor what lies behind a length reaches it.  Blocks of the statistics take `rows` tokens of one document, and
// leave the largest square of them for the document's CTAs to go through: those of dO at the block's first query, those of
// V at kPlaces places for every query of the document (where its keys are more than that, a block takes several turns: one
// query over 65,501 keys, 1131 us; with 8 places 2337).
constexpr int kPlaces = 64;
struct Stat {
    int q_rows, k_rows;      // tokens of a block
    int64_t q_blocks;        // blocks of queries, before those of keys
    float2* stat;            // [Hq][Tq] lse log2 e (infinite for empty rows), delta
    float* norms;            // [Tq] of dO, [kPlaces Tq] of V
};

__host__ __device__ __forceinline__ int stat_rows(int heads) { return heads >= 16 ? 8 : 128 / heads; }

__device__ __forceinline__ int64_t stat_places(const Span& s, int k_rows) {
    return min((int64_t)(s.lk + k_rows - 1) / k_rows, kPlaces * (int64_t)s.lq);
}

struct Grad {
    Attn a;
    float scale;
    Stat st;
    void *dq, *dk, *dv;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;      // of dq, dk, dv
    int key_blocks;
};

struct Heads {
    const void* p;
    int64_t tok, head;
};

// The document of block t where documents have a block for every `rows` tokens begun, and one more at most; and which of its
// blocks that is.
__device__ __forceinline__ int stat_block(const int32_t* cu, int docs, int rows, int64_t t, int64_t* which) {
    int lo = 0, hi = docs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if ((int64_t)(cu[mid] / rows) + mid <= t) lo = mid;
        else hi = mid;
    }
    *which = t - ((int64_t)(cu[lo] / rows) + lo);
    return lo;
}

template <typename T, int DP>
__global__ void __launch_bounds__(256)
    k_attn_stat(const Heads dout, const Heads o, const float* __restrict__ lse, const Heads v, const __grid_constant__ Attn a,
                const __grid_constant__ Stat st) {
    pdl_begin();
    constexpr int G = DP / 8, kRows = 256 / G;            // lanes a row
    const int gl = threadIdx.x % G, own = threadIdx.x / G;
    const bool in = 8 * gl < a.D;
    const bool keys = blockIdx.x >= st.q_blocks;
    const int rows = keys ? st.k_rows : st.q_rows;
    if (blockIdx.x == 0)                                  // also those without a tile that some block works on
        for (int d = threadIdx.x; d < a.docs; d += 256) report_span(a, d, INT32_MAX);
    int64_t which = blockIdx.x;
    Span sp{0, (int)a.Tq};                                // bf16 has no use for documents here
    if constexpr (Elem<T>::kFmt == 0)
        sp = span_of(a, stat_block(keys ? a.cu_k : a.cu_q, a.docs, rows, keys ? blockIdx.x - st.q_blocks : blockIdx.x, &which));
    const int64_t places = keys ? stat_places(sp, rows) : (sp.lq + rows - 1) / rows;
    if (which < 0 || which >= places) return;
    float big = 0.0f;
    constexpr int U = 4;                                  // rows on their way at once
    if (!keys) {
        const int t0 = (int)which * rows, n = min(rows, sp.lq - t0) * a.Hq;
        for (int r0 = 0; r0 < n; r0 += kRows * U) {
            uint4 xs[U], ys[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * kRows + own, h = r % a.Hq;
                const int64_t t = sp.q0 + t0 + r / a.Hq;
                xs[u] = ys[u] = make_uint4(0, 0, 0, 0);
                if (r < n && in) {
                    xs[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(dout.p) + t * dout.tok + h * dout.head + 8 * gl);
                    ys[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(o.p) + t * o.tok + h * o.head + 8 * gl);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * kRows + own, h = r % a.Hq;
                const int64_t t = sp.q0 + t0 + r / a.Hq;
                const uint32_t xw[4] = {xs[u].x, xs[u].y, xs[u].z, xs[u].w}, yw[4] = {ys[u].x, ys[u].y, ys[u].z, ys[u].w};
                float dot = 0.0f, sq = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = Elem<T>::unpack(xw[i]), y = Elem<T>::unpack(yw[i]);
                    dot += x.x * y.x + x.y * y.y;
                    sq += x.x * x.x + x.y * x.y;
                }
#pragma unroll
                for (int x = G / 2; x > 0; x >>= 1) {
                    dot += __shfl_xor_sync(0xffffffffu, dot, x);
                    if constexpr (Elem<T>::kFmt == 0) sq += __shfl_xor_sync(0xffffffffu, sq, x);
                }
                if (sq < INFINITY) big = fmaxf(big, sq);
                if (r < n && gl == 0) {
                    const float l = lse[(int64_t)h * a.Tq + t];
                    st.stat[h * a.Tq + t] = make_float2(l == -INFINITY ? INFINITY : l * kLog2e, dot);
                }
            }
        }
    } else {
        for (int64_t t0 = which * rows; t0 < sp.lk; t0 += places * rows) {
            const int n = (int)min((int64_t)rows, sp.lk - t0) * a.Hk;
            for (int r0 = 0; r0 < n; r0 += kRows * U) {
                uint4 xs[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = r0 + u * kRows + own;
                    const int64_t t = sp.k0 + t0 + r / a.Hk;
                    xs[u] = make_uint4(0, 0, 0, 0);
                    if (r < n && in) xs[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(v.p) + t * v.tok + r % a.Hk * v.head + 8 * gl);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t xw[4] = {xs[u].x, xs[u].y, xs[u].z, xs[u].w};
                    float sq = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 y = Elem<T>::unpack(xw[i]);
                        sq += y.x * y.x + y.y * y.y;
                    }
#pragma unroll
                    for (int x = G / 2; x > 0; x >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, x);
                    if (sq < INFINITY) big = fmaxf(big, sq);
                }
            }
        }
    }
    if constexpr (Elem<T>::kFmt == 0) {
        __shared__ float sm[8];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
        if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = big;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int i = 1; i < 8; ++i) big = fmaxf(big, sm[i]);
            st.norms[keys ? a.Tq + kPlaces * (int64_t)sp.q0 + which : sp.q0 + which] = big;
        }
    }
}

// A compute warpgroup takes 32 streamed columns: rows this short leave registers for two (heads up to 64) or four
// warpgroups a CTA, and 16 compute warps on every SM.  Heads up to 64 stream tiles of 64, two CTAs a SM: one's softmax runs
// under the other's products, starts and ends.  Wider heads leave tensor memory for one CTA, with tiles of 128.
template <int DP>
struct Bwd {
    static constexpr int kGroups = DP == 64 ? 2 : 4;          // compute warpgroups, 32 streamed rows each
    static constexpr int kCtas = DP == 64 ? 2 : 1;
    static constexpr int kBT = 32 * kGroups;
    static constexpr int kThreads = 128 * kGroups + 64;       // then the loader and the MMA issuer
    static constexpr int kStages = DP == 64 ? 4 : 2;
    static constexpr int kTile = 128 * DP * 2;                // stationary
    static constexpr int kStrip = kBT * 128;                  // 64 values of every streamed row
    static constexpr int kPart = kStrip * (DP / 64);          // a streamed tile
    static constexpr int kStream = 2 * kTile;                 // offset of the ring
    static constexpr int kStats = kStream + kStages * 2 * kPart;
    static constexpr int kStatRoom = kBT * 8;
    static constexpr int kBars = kStats + kStages * kStatRoom;
    static constexpr int kSmem = kBars + 256;
    static constexpr uint32_t kCols = DP == 64 ? 256 : 512;   // tensor memory
    static constexpr uint32_t kS = 0, kDP = kBT, kOut0 = 2 * kBT, kOut1 = 2 * kBT + DP;
};

struct Bars {
    uint64_t *a_full, *b_full, *b_empty, *s_full, *dp_full, *p_full, *ds_full, *done, *drain;
    volatile int* abort_flag;
};

// log2 of the factor that P carries before it is rounded.
template <typename T> constexpr float kPLift = 0.0f;
template <> constexpr float kPLift<__half> = 15.0f;

// The factor that a document's dS carries before it is rounded.
template <typename T>
__device__ __forceinline__ float ds_lift(const Stat& st, const Span& sp, int64_t Tq) {
    if constexpr (Elem<T>::kFmt == 1) {
        return 1.0f;
    } else {
        const int lane = threadIdx.x & 31;
        const float *of_do = st.norms + sp.q0, *of_v = st.norms + Tq + kPlaces * (int64_t)sp.q0;
        const int64_t n_do = (sp.lq + st.q_rows - 1) / st.q_rows, n_v = stat_places(sp, st.k_rows);
        float a = 0.0f, b = 0.0f;
        for (int64_t i = lane; i < n_do; i += 32) a = fmaxf(a, of_do[i]);
        for (int64_t i = lane; i < n_v; i += 32) b = fmaxf(b, of_v[i]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, x));
            b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, x));
        }
        // log2 (2 max|dO| max|V|) = 1 + (log2 a + log2 b) / 2
        const float l = 1.0f + 0.5f * (log2f(a) + log2f(b));
        return a > 0.0f && b > 0.0f ? exp2f(fminf(fmaxf(floorf(14.0f - l), -60.0f), 60.0f)) : 1.0f;
    }
}

template <typename T, int DP, bool KEYS, bool CAP, bool BIAS>
__device__ __forceinline__ void grad_cta(const CUtensorMap& ma0, const CUtensorMap& ma1, const CUtensorMap& mb0,
                                         const CUtensorMap& mb1, const Grad& g, uint8_t* smem, const Bars& b,
                                         uint32_t tmem, int block, int doc, int tile) {
    using C = Bwd<DP>;
    const Attn& a = g.a;
    volatile int* abort_flag = b.abort_flag;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const Span sp = span_of(a, doc);
    const int off = sp.lk - sp.lq;
    const int head = KEYS ? 0 : block % a.Hq;                       // query CTAs: their head
    const int kvh = KEYS ? block % a.Hk : head / a.group;
    const int r0 = tile * 128;                                      // first stationary row within the document
    // streamed tiles: queries t0 .. t1 - 1 of each head of the group, or keys
    int t0 = 0, t1 = 0;
    if (KEYS) {
        if (r0 < sp.lk) {
            t1 = (sp.lq + C::kBT - 1) / C::kBT;
            if (a.causal && r0 >= sp.prefix) t0 = min(t1, max(0, r0 - off) / C::kBT);
        }
    } else {
        t1 = (key_end(a, sp, r0 + 128) + C::kBT - 1) / C::kBT;
    }
    const int per = t1 - t0, total = KEYS ? per * a.group : per;

    if (warp == 4 * C::kGroups) {
        if (total > 0) {
            bool ok = true;
            const int row = (KEYS ? sp.k0 : sp.q0) + r0, h = KEYS ? kvh : head;
            if (lane == 0) {
                mbar_arrive_expect_tx(b.a_full, 2 * C::kTile);
#pragma unroll
                for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                    for (int r = 0; r < 128; r += 64) {
                        tma_tile3d(smem_u32(smem + c * 16384 + r * 128), &ma0, 64 * c, h, row + r, b.a_full);
                        tma_tile3d(smem_u32(smem + C::kTile + c * 16384 + r * 128), &ma1, 64 * c, h, row + r, b.a_full);
                    }
            }
            // each lane's share of a tile's statistics, fetched a tile ahead
            float2 stat[C::kBT / 32];
            auto fetch = [&](int t, int bh) {
#pragma unroll
                for (int e = 0; e < C::kBT / 32; ++e) {
                    const int64_t at = sp.q0 + (int64_t)C::kBT * t + lane + 32 * e;
                    stat[e] = at < a.Tq ? g.st.stat[bh * a.Tq + at] : make_float2(0.0f, 0.0f);
                }
            };
            int t = t0, bh = KEYS ? kvh * a.group : kvh;
            if (KEYS) fetch(t, bh);
            for (int i = 0; i < total; ++i) {
                const int st = i % C::kStages;
                ok = __all_sync(0xffffffffu, wait_bar(b.b_empty + st, ((i / C::kStages) & 1u) ^ 1u, abort_flag));
                if (!ok) break;
                const int brow = (KEYS ? sp.q0 : sp.k0) + C::kBT * t;
                if (lane == 0) {
                    uint8_t* to = smem + C::kStream + st * 2 * C::kPart;
                    mbar_arrive_expect_tx(b.b_full + st, 2 * C::kPart);
#pragma unroll
                    for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                        for (int r = 0; r < C::kBT; r += 64) {
                            tma_tile3d(smem_u32(to + c * C::kStrip + r * 128), &mb0, 64 * c, bh, brow + r, b.b_full + st);
                            tma_tile3d(smem_u32(to + C::kPart + c * C::kStrip + r * 128), &mb1, 64 * c, bh, brow + r, b.b_full + st);
                        }
                }
                if (KEYS) {
                    float* to = reinterpret_cast<float*>(smem + C::kStats + st * C::kStatRoom);
#pragma unroll
                    for (int e = 0; e < C::kBT / 32; ++e) {
                        to[lane + 32 * e] = kPLift<T> - stat[e].x;
                        to[C::kBT + lane + 32 * e] = -stat[e].y;
                    }
                }
                mbar_arrive(b.b_full + st);
                if (++t == t1) {
                    t = t0;
                    ++bh;
                }
                if (KEYS && i + 1 < total) fetch(t, bh);
            }
            if (!ok && lane == 0) {
                *abort_flag = 1;
                flag(a.status, PMG_ERR_TIMEOUT);
            }
        }
    } else if (warp == 4 * C::kGroups + 1) {
        const int ksteps = (a.D + 15) / 16;
        const uint32_t id_s = idesc16(Elem<T>::kFmt, 128, C::kBT, false, false);
        const uint32_t id_o = idesc16(Elem<T>::kFmt, 128, ksteps * 16, false, true);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) { return (bool)__all_sync(0xffffffffu, wait_bar(bar, ph, abort_flag)); };
        auto stage = [&](int i) { return smem + C::kStream + (i % C::kStages) * 2 * C::kPart; };
        // a streamed tile has landed; rows behind the document's last must not reach a sum over rows (0 * NaN)
        int lt = t0;                                    // tile of the next call
        auto landed = [&](int i) {
            if (!wait(b.b_full + i % C::kStages, (i / C::kStages) & 1u)) return false;
            const int valid = (KEYS ? sp.lq : sp.lk) - C::kBT * lt;
            if (++lt == t1) lt = t0;
            if (valid < C::kBT) {
                uint8_t* s = stage(i);
                for (int c = 0; c < (KEYS ? 2 : 1) * (DP / 64); ++c)
                    for (int x = valid * 128 + lane * 16; x < C::kStrip; x += 512)
                        *reinterpret_cast<uint4*>(s + c * C::kStrip + x) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
                __syncwarp();
            }
            return true;
        };
        const uint32_t lead = elect_one();
        auto square = [&](int i, int which) {           // scores (0) or dP (1) of tile i
            tc_fence_after();
            const uint32_t x = desc_lo(smem_u32(smem + which * C::kTile), 16), y = desc_lo(smem_u32(stage(i) + which * C::kPart), 16);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
                if (s < ksteps) {
                    const uint32_t in = (s & 3) * 2;
                    mma16(lead, tmem + (which ? C::kDP : C::kS), x + (s >> 2) * 1024 + in, y + (s >> 2) * (C::kStrip / 16) + in, id_s, s > 0);
                }
            mma_commit_if(lead, which ? b.dp_full : b.s_full);
        };
        auto sum = [&](int i, int which) {              // out0 += dS B0, out1 += P B1
            tc_fence_after();
            const uint32_t x = tmem + (which ? C::kS : C::kDP), y = desc_lo(smem_u32(stage(i) + which * C::kPart), C::kStrip);
#pragma unroll
            for (int s = 0; s < C::kBT / 16; ++s)       // each warpgroup's half lies in its own columns
                mma16_ts(lead, tmem + (which ? C::kOut1 : C::kOut0), x + (s >> 1) * 32 + (s & 1) * 8, y + s * 128, id_o, i > 0 || s > 0);
        };
        if (total > 0) {
            ok = wait(b.a_full, 0) && landed(0);
            if (ok) {
                square(0, 0);
                square(0, 1);
            }
            for (int i = 0; i < total && ok; ++i) {
                ok = wait(b.p_full, i & 1u);
                if (!ok) break;
                if (KEYS) sum(i, 1);
                if (i + 1 < total) {
                    ok = landed(i + 1);
                    if (!ok) break;
                    square(i + 1, 0);
                }
                ok = wait(b.ds_full, i & 1u);
                if (!ok) break;
                sum(i, 0);
                mma_commit_if(lead, b.b_empty + i % C::kStages);
                if (i + 1 < total) square(i + 1, 1);
            }
            if (ok) mma_commit_if(lead, b.done);
            if (lane == 0) {
                if (!ok) flag(a.status, PMG_ERR_TIMEOUT);
                if (!ok || *abort_flag) {
                    *abort_flag = 1;
                    drain_mma(b.drain);
                }
            }
            __syncwarp();
        }
    } else {
        const int w = warp >> 2, row = r0 + (warp & 3) * 32 + lane;        // column half; stationary row in the document
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + C::kS + 32 * w, td = tmem + lanes + C::kDP + 32 * w;
        const float lift = ds_lift<T>(g.st, sp, a.Tq);
        const float pd = Elem<T>::kFmt == 0 ? lift * exp2f(-kPLift<T>) : 1.0f;
        const float c = BIAS ? 1.0f : (CAP ? a.cap2 : a.scale2);
        // columns [lo, hi) of the streamed side take part in this row
        int lo = 0, hi;
        if (KEYS) {
            hi = sp.lq;
            if (a.causal && row >= sp.prefix) lo = max(0, row - off);
        } else {
            hi = last_key(a, sp, row) + 1;
        }
        const bool live = row < (KEYS ? sp.lk : sp.lq);
        const int lo_max = __reduce_max_sync(0xffffffffu, live ? lo : 0), hi_min = __reduce_min_sync(0xffffffffu, live ? hi : INT32_MAX);
        float my_lse = INFINITY, my_delta = 0.0f;
        if (!KEYS && live && sp.q0 + (int64_t)row < a.Tq) {
            const float2 s = g.st.stat[head * a.Tq + sp.q0 + row];
            my_lse = s.x;
            my_delta = s.y;
        }
        const uint64_t my_shift = pack2(kPLift<T> - my_lse, kPLift<T> - my_lse), my_less = pack2(-my_delta, -my_delta);
        bool ok = true;
        int t = t0, h = KEYS ? kvh * a.group : head;
        float slope = BIAS ? a.slopes[h] * kLog2e : 0.0f;
        for (int i = 0; i < total; ++i) {
            const int c0 = C::kBT * t + 32 * w;                            // first column within the document
            const float far = KEYS ? (float)(row - off - c0) : (float)(row + off - c0);
            const bool masked = c0 < lo_max || c0 + 32 > hi_min;
            const float* shift = reinterpret_cast<const float*>(smem + C::kStats + (i % C::kStages) * C::kStatRoom) + 32 * w;
            const float* less = shift + C::kBT;
            auto four = [](const float* at) { return *reinterpret_cast<const ulonglong2*>(at); };   // columns
            if (KEYS) TOK_WAIT(b.b_full + i % C::kStages, (i / C::kStages) & 1u);
            if (!ok) break;
            TOK_WAIT(b.s_full, i & 1u);
            if (!ok) break;
            tc_fence_after();
            float p[32], u[CAP ? 32 : 1];
            uint32_t r[16];
            tmem_ld32(ts, reinterpret_cast<uint32_t*>(p));
            tmem_wait_ld();
            if constexpr (CAP) {
                // rows and columns that take no part do not choose tanh's form
                tanh_scores<32>(a, p, !masked && tanh_fast(a, live ? largest<32>(p) : 0.0f));
#pragma unroll
                for (int k = 0; k < 32; ++k) u[k] = fmaf(-p[k], p[k], 1.0f);             // the cap's slope
            }
            if (BIAS) bias_scores<32>(p, CAP ? a.cap2 : a.scale2, slope, far);
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
                ulonglong2 z = make_ulonglong2(my_shift, my_shift);
                if (KEYS) z = four(shift + k);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint64_t y = fma2(pack2(p[k + 2 * e], p[k + 2 * e + 1]), pack2(c, c), e ? z.y : z.x);
                    const float2 f = unpack2(takes_poly(k / 2 + e, CAP ? 0 : 5) ? ex2_poly(y) : ex2_pair(y));
                    p[k + 2 * e] = f.x;
                    p[k + 2 * e + 1] = f.y;
                }
            }
            if (masked) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    if (c0 + k < lo || c0 + k >= hi) p[k] = 0.0f;
            }
            if (KEYS) {
#pragma unroll
                for (int k = 0; k < 16; ++k) r[k] = Elem<T>::pack(p[2 * k], p[2 * k + 1]);
                tmem_st16(ts, r);                         // over scores that this warp has read
                tmem_wait_st();
            }
            tc_fence_before();
            mbar_arrive(b.p_full);
            if constexpr (CAP) {
#pragma unroll
                for (int k = 0; k < 32; ++k) p[k] *= u[k];
            }
            TOK_WAIT(b.dp_full, i & 1u);
            if (!ok) break;
            tc_fence_after();
            float d[32];
            tmem_ld32(td, reinterpret_cast<uint32_t*>(d));
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
                ulonglong2 z = make_ulonglong2(my_less, my_less);
                if (KEYS) z = four(less + k);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int at = k + 2 * e;
                    uint64_t y = mul2(add2(pack2(d[at], d[at + 1]), e ? z.y : z.x), pack2(p[at], p[at + 1]));
                    if (Elem<T>::kFmt == 0) y = mul2(y, pack2(pd, pd));
                    const float2 f = unpack2(y);
                    d[at] = f.x;
                    d[at + 1] = f.y;
                }
            }
            if (masked) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    if (c0 + k < lo || c0 + k >= hi) d[k] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = Elem<T>::pack(d[2 * k], d[2 * k + 1]);
            tmem_st16(td, r);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(b.ds_full);
            if (++t == t1) {                              // the next head of the group
                t = t0;
                ++h;
                if (BIAS && i + 1 < total) slope = a.slopes[h] * kLog2e;
            }
        }
        if (ok && total > 0) TOK_WAIT(b.done, 0);
        if (ok) {
            tc_fence_after();
            const float f0 = g.scale / lift, f1 = Elem<T>::kFmt == 0 ? exp2f(-kPLift<T>) : 1.0f;
            const int room = KEYS ? sp.room : sp.lq;        // rows behind k_len get zeros
            const int64_t at = (KEYS ? sp.k0 : sp.q0) + (int64_t)row;
            const bool mine = row < room && at < (KEYS ? a.Tk : a.Tq);
            const bool zero = total == 0 || !live;
#pragma unroll
            for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
                T* base = KEYS ? static_cast<T*>(which ? g.dv : g.dk) + at * (which ? g.v_tok : g.k_tok) + kvh * (which ? g.v_head : g.k_head)
                               : static_cast<T*>(g.dq) + at * g.q_tok + head * g.q_head;
                const float f = which ? f1 : f0;
                {
                    const int c1 = 32 * w;                                  // a group's share of the columns: DP = 32 groups
                    float v[32];
                    if (total > 0) {
                        tmem_ld32(tmem + lanes + (which ? C::kOut1 : C::kOut0) + c1, reinterpret_cast<uint32_t*>(v));
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = zero ? 0.0f : v[k] * f;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (mine && c1 + 8 * k < a.D)
                            *reinterpret_cast<uint4*>(base + c1 + 8 * k) =
                                make_uint4(Elem<T>::pack(v[8 * k], v[8 * k + 1]), Elem<T>::pack(v[8 * k + 2], v[8 * k + 3]),
                                           Elem<T>::pack(v[8 * k + 4], v[8 * k + 5]), Elem<T>::pack(v[8 * k + 6], v[8 * k + 7]));
                }
            }
        } else if (lane == 0) {
            *abort_flag = 1;
            flag(a.status, PMG_ERR_TIMEOUT);
        }
    }
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(Bwd<DP>::kThreads, Bwd<DP>::kCtas)
    k_attn_grad(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo, const __grid_constant__ Grad g) {
    using C = Bwd<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars b;
    b.a_full = reinterpret_cast<uint64_t*>(smem + C::kBars);
    b.b_full = b.a_full + 1;
    b.b_empty = b.b_full + C::kStages;
    b.s_full = b.b_empty + C::kStages;
    b.dp_full = b.s_full + 1;
    b.p_full = b.dp_full + 1;
    b.ds_full = b.p_full + 1;
    b.done = b.ds_full + 1;
    b.drain = b.done + 1;
    uint32_t* slot = reinterpret_cast<uint32_t*>(b.drain + 1);
    b.abort_flag = reinterpret_cast<volatile int*>(slot + 1);
    int* where = reinterpret_cast<int*>(slot + 2);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const bool keys = (int)blockIdx.x < g.key_blocks;
    const int block = keys ? blockIdx.x : blockIdx.x - g.key_blocks;

    if (threadIdx.x == 0) {
        mbar_init(b.a_full, 1);
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(b.b_full + i, 33);             // the bytes, and the loader's lanes with the statistics
            mbar_init(b.b_empty + i, 1);
        }
        mbar_init(b.s_full, 1);
        mbar_init(b.dp_full, 1);
        mbar_init(b.p_full, 128 * C::kGroups);
        mbar_init(b.ds_full, 128 * C::kGroups);
        mbar_init(b.done, 1);
        mbar_init(b.drain, 1);
        *b.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 4 * C::kGroups + 1) tmem_alloc(slot, C::kCols);
    pdl_begin();
    if (warp == 4 * C::kGroups) {
        int doc = -1, tile = 0;
        const int32_t* cu = keys ? g.a.cu_k : g.a.cu_q;
        const int t = block / (keys ? g.a.Hk : g.a.Hq);
        bool found;
        if (g.a.causal) {                // the first keys are seen by most queries, the last queries see most keys
            found = find_level(cu, g.a.docs, 128, t, &doc, &tile);
            if (found && !keys) tile = (max(0, cu[doc + 1] - cu[doc]) + 127) / 128 - 1 - tile;
        } else {
            found = find_tile(cu, g.a.docs, 128, t, &doc, &tile);
        }
        if (lane == 0) {
            where[0] = found ? doc : -1;
            where[1] = tile;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *slot, 0);
    if (where[0] >= 0) {
        if (keys) grad_cta<T, DP, true, CAP, BIAS>(mk, mv, mq, mdo, g, smem, b, tmem, block, where[0], where[1]);
        else grad_cta<T, DP, false, CAP, BIAS>(mq, mdo, mk, mv, g, smem, b, tmem, block, where[0], where[1]);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 4 * C::kGroups + 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kCols);
    }
}

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

struct Ins {
    Heads dout, o, q, k, v;
    const float* lse;
    float* ws;
};

template <typename T, int DP, bool CAP, bool BIAS>
int run(Grad g, const Ins& in, cudaStream_t s) {
    using C = Bwd<DP>;
    const Attn& a = g.a;
    const int rc = raise_smem<k_attn_grad<T, DP, CAP, BIAS>>(C::kSmem);
    if (rc != PMG_OK) return rc;
    g.st.q_rows = stat_rows(a.Hq);
    g.st.k_rows = stat_rows(a.Hk);
    const bool by_document = Elem<T>::kFmt == 0;
    g.st.q_blocks = by_document ? a.Tq / g.st.q_rows + a.docs : (a.Tq + g.st.q_rows - 1) / g.st.q_rows;
    g.st.stat = reinterpret_cast<float2*>(in.ws);
    g.st.norms = in.ws + 2 * a.Tq * a.Hq;
    const int64_t stat_blocks = g.st.q_blocks + (by_document ? a.Tk / g.st.k_rows + a.docs : 0);
    if (stat_blocks > INT32_MAX) return PMG_ERR_UNSUPPORTED;
    k_attn_stat<T, DP><<<(unsigned)stat_blocks, 256, 0, s>>>(in.dout, in.o, in.lse, in.v, a, g.st);
    PMG_LAUNCH_CHECK();
    const int64_t key_blocks = (a.Tk / 128 + a.docs) * a.Hk, query_blocks = (a.Tq / 128 + a.docs) * a.Hq;
    if (key_blocks + query_blocks > INT32_MAX) return PMG_ERR_UNSUPPORTED;
    g.key_blocks = (int)key_blocks;
    CUtensorMap mq, mk, mv, mdo;
    int e = head_map(&mq, in.q.p, in.q.tok, in.q.head, a.Tq, a.Hq, a.D, 64);
    if (e == PMG_OK) e = head_map(&mdo, in.dout.p, in.dout.tok, in.dout.head, a.Tq, a.Hq, a.D, 64);
    if (e == PMG_OK) e = head_map(&mk, in.k.p, in.k.tok, in.k.head, a.Tk, a.Hk, a.D, 64);
    if (e == PMG_OK) e = head_map(&mv, in.v.p, in.v.tok, in.v.head, a.Tk, a.Hk, a.D, 64);
    if (e != PMG_OK) return e;
    return launch_after(k_attn_grad<T, DP, CAP, BIAS>, dim3((unsigned)(key_blocks + query_blocks)), C::kThreads, C::kSmem, s, mq,
                        mk, mv, mdo, g);
}

template <typename T, int DP>
int by_score(const Grad& g, const Ins& in, cudaStream_t s) {
    if (g.a.cap2 > 0.0f) return g.a.slopes ? run<T, DP, true, true>(g, in, s) : run<T, DP, true, false>(g, in, s);
    return g.a.slopes ? run<T, DP, false, true>(g, in, s) : run<T, DP, false, false>(g, in, s);
}

}  // namespace
}  // namespace pmg

using namespace pmg;

extern "C" size_t pmg_attention_grad_workspace_bytes(int64_t Tq, int32_t Hq) {
    if (Tq < 0 || Hq < 0) return 0;
    return (size_t)Tq * (Hq * sizeof(float2) + (1 + kPlaces) * sizeof(float));
}

extern "C" int pmg_attention_grad(const void* dout, int64_t do_tok, int64_t do_head, const void* o, int64_t o_tok,
                                  int64_t o_head, const float* lse, const void* q, int64_t q_tok, int64_t q_head,
                                  const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
                                  int64_t v_head, int32_t dtype, int64_t Tq, int64_t Tk, int32_t Hq, int32_t Hk,
                                  int32_t D, const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_len,
                                  int32_t docs, float scale, int32_t causal, const int32_t* prefix, float softcap,
                                  const float* slopes, void* dq, int64_t dq_tok, int64_t dq_head, void* dk,
                                  int64_t dk_tok, int64_t dk_head, void* dv, int64_t dv_tok, int64_t dv_head,
                                  void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
    Grad g{};
    const int rc = fill_attn(&g.a, dtype, cu_q, cu_k, k_len, docs, Tq, Tk, Hq, Hk, D, scale, causal, prefix, softcap, slopes, status);
    if (rc != PMG_OK) return rc;
    auto ok = [](const void* p, int64_t t, int64_t h) { return p && !(reinterpret_cast<uintptr_t>(p) & 15) && !(t & 7) && !(h & 7); };
    cudaStream_t s = as_stream(stream);
    // without queries or keys every gradient that has rows is zero
    if (docs == 0 || Tq == 0 || Tk == 0) {
        if (Tq > 0 && (!ok(dq, dq_tok, dq_head) || dq_head != D || dq_tok != (int64_t)Hq * D)) return PMG_ERR_BAD_ARG;
        if (Tk > 0 && (!ok(dk, dk_tok, dk_head) || dk_head != D || dk_tok != (int64_t)Hk * D || !ok(dv, dv_tok, dv_head) ||
                       dv_head != D || dv_tok != (int64_t)Hk * D))
            return PMG_ERR_BAD_ARG;
        if (Tq > 0) PMG_CUDA_TRY(cudaMemsetAsync(dq, 0, (size_t)Tq * Hq * D * 2, s));
        if (Tk > 0) PMG_CUDA_TRY(cudaMemsetAsync(dk, 0, (size_t)Tk * Hk * D * 2, s));
        if (Tk > 0) PMG_CUDA_TRY(cudaMemsetAsync(dv, 0, (size_t)Tk * Hk * D * 2, s));
        return PMG_OK;
    }
    if (!lse || !ok(dout, do_tok, do_head) || !ok(o, o_tok, o_head) || !ok(q, q_tok, q_head) || !ok(k, k_tok, k_head) ||
        !ok(v, v_tok, v_head) || !ok(dq, dq_tok, dq_head) || !ok(dk, dk_tok, dk_head) || !ok(dv, dv_tok, dv_head))
        return PMG_ERR_BAD_ARG;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < pmg_attention_grad_workspace_bytes(Tq, Hq))
        return PMG_ERR_BAD_ARG;
    g.scale = scale;
    g.dq = dq; g.dk = dk; g.dv = dv;
    g.q_tok = dq_tok; g.q_head = dq_head; g.k_tok = dk_tok; g.k_head = dk_head; g.v_tok = dv_tok; g.v_head = dv_head;
    const Ins in{{dout, do_tok, do_head}, {o, o_tok, o_head}, {q, q_tok, q_head}, {k, k_tok, k_head}, {v, v_tok, v_head}, lse,
                 static_cast<float*>(workspace)};
    if (dtype == PMG_BF16) return D <= 64 ? by_score<__nv_bfloat16, 64>(g, in, s) : by_score<__nv_bfloat16, 128>(g, in, s);
    return D <= 64 ? by_score<__half, 64>(g, in, s) : by_score<__half, 128>(g, in, s);
}
