// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its gradient.
//
//   n = x / sqrt(mean(x^2) + eps) * w        over the D values of one head of one token
//   y = R(p) n                               pairs (a, b) -> (a cos - b sin, b cos + a sin), angles of position p
//
// Pairs are (i, i + rot/2) or, interleaved, (2i, 2i + 1), among the first rot values; the others pass through.
// Backwards, with g = R(p)^T dy and n' = x r, r = 1 / sqrt(mean(x^2) + eps):
//   dw = sum over tokens and heads of g n',   dx = r (g w - n' mean(g w n')).
//
// Bound by HBM: forwards one read and one write of q and k, backwards two reads and one write.  A group of lanes owns a
// row (D values, 16 bytes a lane) and walks all heads of one token with that token's angles in registers: the angles are 8
// bytes per pair against 2 bytes per value, so loading them per head would cost more first-level cache traffic than the
// heads themselves (four heads an item: 72 us and more for the first size below).  A block works on queries or on keys, so
// that the weights stay in registers too.  Where pairs are (i, i + rot/2) a lane holds V/2 values on either side: the
// exchange that one run of V values a lane needs took 54 us.  Two heads are worked on while the next two are on their way.
// Measured: 38,400 tokens, 16 + 4 heads of 64, bf16: 44 us (4.5 TB/s of 6.5; copying as much takes 31), in fp32 75 to 79 us
// (5.0 to 5.2 TB/s), backwards 124; backwards 19,201 tokens, 16 + 4 heads of 128, fp16: 78 us (3.8 TB/s).
// Sums and norms are fp32; a value is rounded once, when it is stored.
#include <algorithm>

#include "tok_common.cuh"

namespace pmg {
namespace {

constexpr int kThreads = 256;                         // a block's, backwards and for the general form
constexpr int kMaxD = 256;

struct Side {                 // queries or keys
    const void* x;
    const void* dy;
    void* out;
    const float* w;
    int64_t xt, xh, yt, yh, ot, oh;   // strides of x, dy, out in elements: token, head
    int H;
};

struct RopeArgs {
    Side side[2];
    const float *cos, *sin;
    const int32_t* pos;
    int64_t T;
    int places, D, half, interleaved, heads[2], chunks[2], blocks[2];   // heads per item, items per token, blocks of each side
    float eps;
    int32_t* status;
    float* part;              // gradients of w: [blocks[0] + blocks[1]][D]
};

// A vector of V values of a row (16 or 8 bytes of 16-bit values, 16 bytes of fp32 ones) and its pairs in fp32.
template <typename T, int V>
struct Row {
    static constexpr int kWords = V * (int)sizeof(T) / 4;
    uint32_t w[kWords];
    // from one place, or its halves from two
    template <bool WHOLE>
    __device__ __forceinline__ void get(const T* p, const T* q) {
        if constexpr (WHOLE && kWords == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (kWords == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(p), v = *reinterpret_cast<const uint2*>(q);
            w[0] = u.x; w[1] = u.y; w[2] = v.x; w[3] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
            w[1] = *reinterpret_cast<const uint32_t*>(q);
        }
    }
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return tok::Elem<T>::unpack(w[i]);
    }
    __device__ __forceinline__ void set(int i, float2 f) {
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(f.x);
            w[2 * i + 1] = __float_as_uint(f.y);
        } else {
            w[i] = tok::Elem<T>::pack(f.x, f.y);
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void put(T* p, T* q) const {
        if constexpr (WHOLE && kWords == 4) {
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if constexpr (kWords == 4) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            *reinterpret_cast<uint2*>(q) = make_uint2(w[2], w[3]);
        } else {
            *reinterpret_cast<uint32_t*>(p) = w[0];
            *reinterpret_cast<uint32_t*>(q) = w[1];
        }
    }
};

__device__ __forceinline__ uint64_t two(float2 f) { return tok::pack2(f.x, f.y); }
__device__ __forceinline__ float2 swapped(float2 f) { return make_float2(f.y, f.x); }

// The position of token t; one outside the table is reported and taken as 0.
__device__ __forceinline__ int64_t place_of(const RopeArgs& a, int64_t t, bool tell) {
    const int p = a.pos ? a.pos[t] : (int)t;
    if (p >= 0 && p < a.places) return p;
    if (tell) flag(a.status, PMG_ERR_RANGE);
    return 0;
}

// G lanes a row, V values a lane, pairs of them in the packed fp32 pipe; U heads at once, the next U on their way.
// IL: interleaved pairs, which lie within a lane's vector.  What bounds this after HBM is the chain of a row, so warps count:
// forwards 28 a SM in blocks of four (72 registers) 43 us, 16 of them with four heads in flight 47, 32 of 64 registers, which
// spill, 45; backwards 16 a SM in blocks of eight (128 registers) 78 us, 8 of them 106, 24 with one head in flight 90.
template <bool GRAD> constexpr int kBlock = GRAD ? kThreads : 128;
template <typename T, int V, int U, bool GRAD, bool IL>
__global__ void __launch_bounds__(kBlock<GRAD>, GRAD ? 2 : 7) k_qk_norm_rope(const __grid_constant__ RopeArgs a, int G) {
    using namespace tok;
    using R = Row<T, V>;
    constexpr int NP = V / 2;
    auto partner = [](int i) { return IL ? i : (i + NP / 2) % NP; };        // the packed pair with a pair's other sides
    pdl_begin();
    extern __shared__ float sm[];
    const int lane = threadIdx.x & 31, per_warp = 32 / G, gi = lane / G, gl = lane % G;
    const int which = (int)blockIdx.x >= a.blocks[0];
    const Side& s = a.side[which];
    const int per_token = a.chunks[which], heads = a.heads[which];
    const int64_t items = a.T * per_token;
    const int64_t first = (int64_t)(blockIdx.x - (which ? a.blocks[0] : 0)) * (kBlock<GRAD> / 32) + (threadIdx.x >> 5);
    const int64_t stride = (int64_t)a.blocks[which] * (kBlock<GRAD> / 32) * per_warp;
    const float inv_d = 1.0f / (float)a.D;
    const bool in = gl * V < a.D;
    // A lane's values: V / 2 from `at` on and V / 2 from `bt` on.  They are one run, except where the pairs are (i, i +
    // rot/2): there a turned lane holds both sides of its pairs, and nothing has to be exchanged.
    constexpr int HV = V / 2;
    const bool turned = IL ? gl * V < 2 * a.half : gl * HV < a.half;
    const int ang = gl * HV;
    const int at = !in ? 0 : IL || !turned ? gl * V : gl * HV;
    const int bt = !in ? 0 : IL || !turned ? at + HV : at + a.half;
    const int ab = bt - at;
    uint64_t w2[NP], acc[GRAD ? NP : 1];                // the weights
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = i < NP / 2 ? at + 2 * i : bt + 2 * i - HV;
        w2[i] = s.w ? pack2(s.w[c], s.w[c + 1]) : pack2(1.0f, 1.0f);
        if constexpr (GRAD) acc[i] = 0;
    }

    // A token's angles are two dependent loads away: its position is fetched two items ahead, its angles one.
    constexpr int NA = V / 4;
    float2 fc[NA], fs[NA];
    auto token = [&](int64_t base) {
        const int64_t item = min(base + gi, items - 1);
        return per_token == 1 ? item : item / per_token;
    };
    auto angles = [&](int64_t place) {
        if (!turned) return;
#pragma unroll
        for (int e = 0; e < NA; ++e) {
            fc[e] = *reinterpret_cast<const float2*>(a.cos + place * a.half + ang + 2 * e);
            fs[e] = *reinterpret_cast<const float2*>(a.sin + place * a.half + ang + 2 * e);
        }
    };
    int64_t next_place = 0;
    if (first * per_warp < items) {
        angles(place_of(a, token(first * per_warp), gl == 0));
        next_place = place_of(a, token(first * per_warp + stride), gl == 0);
    }

    R rx[2][U] = {}, rd[2][GRAD ? U : 1] = {};          // rows that are not read keep what they held, and count as 0
    for (int64_t base = first * per_warp; base < items; base += stride) {
        const bool live = base + gi < items;
        const int64_t item = live ? base + gi : items - 1;
        const int64_t t = per_token == 1 ? item : item / per_token;
        const int h0 = (int)(item - t * per_token) * heads;
        const int n = live && in ? min(heads, s.H - h0) : 0;
        // where the next head is read and written
        const T* x = reinterpret_cast<const T*>(s.x) + t * s.xt + h0 * s.xh + at;
        const T* d = GRAD ? reinterpret_cast<const T*>(s.dy) + t * s.yt + h0 * s.yh + at : nullptr;
        T* o = reinterpret_cast<T*>(s.out) + t * s.ot + h0 * s.oh + at;
        auto fetch = [&](int b, int h) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (h + u < n) {
                    rx[b][u].template get<IL>(x, x + ab);
                    if constexpr (GRAD) rd[b][u].template get<IL>(d, d + ab);
                }
                x += s.xh;
                if constexpr (GRAD) d += s.yh;
            }
        };
        fetch(0, 0);
        // this token's turn: the rotation's sign in sn, and forwards the weights in both
        uint64_t cs[NP], sn[NP];
        {
            float c[V], z[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                c[e] = 1.0f;
                z[e] = 0.0f;
            }
            if (turned) {
#pragma unroll
                for (int e = 0; e < NA; ++e) {
                    if constexpr (IL) {
                        c[4 * e] = c[4 * e + 1] = fc[e].x;
                        c[4 * e + 2] = c[4 * e + 3] = fc[e].y;
                        z[4 * e] = -fs[e].x;
                        z[4 * e + 1] = fs[e].x;
                        z[4 * e + 2] = -fs[e].y;
                        z[4 * e + 3] = fs[e].y;
                    } else {
                        c[2 * e] = c[HV + 2 * e] = fc[e].x;
                        c[2 * e + 1] = c[HV + 2 * e + 1] = fc[e].y;
                        z[2 * e] = -fs[e].x;
                        z[2 * e + 1] = -fs[e].y;
                        z[HV + 2 * e] = fs[e].x;
                        z[HV + 2 * e + 1] = fs[e].y;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                cs[i] = pack2(c[2 * i], c[2 * i + 1]);
                sn[i] = GRAD ? pack2(-z[2 * i], -z[2 * i + 1]) : pack2(z[2 * i], z[2 * i + 1]);
                if constexpr (!GRAD) {
                    cs[i] = mul2(cs[i], w2[i]);
                    sn[i] = mul2(sn[i], IL ? two(swapped(unpack2(w2[i]))) : w2[partner(i)]);
                }
            }
        }
        if (base + stride < items) {
            angles(next_place);
            next_place = place_of(a, token(base + 2 * stride), gl == 0);
        }
        auto work = [&](int b, int h) {
            uint64_t v[U][NP], g[GRAD ? U : 1][NP];
            float sq[U], gx[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint64_t q2 = 0, x2 = 0;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    v[u][i] = two(rx[b][u].pair(i));
                    q2 = fma2(v[u][i], v[u][i], q2);
                    if constexpr (GRAD) {            // g = R(p)^T dy
                        const float2 y = rd[b][u].pair(i);
                        const uint64_t other2 = two(IL ? swapped(y) : rd[b][u].pair(partner(i)));
                        g[u][i] = fma2(two(y), cs[i], mul2(other2, sn[i]));
                        x2 = fma2(mul2(g[u][i], w2[i]), v[u][i], x2);
                    }
                }
                const float2 f = unpack2(q2), e = unpack2(x2);
                sq[u] = h + u < n ? f.x + f.y : 0.0f;
                gx[u] = h + u < n ? e.x + e.y : 0.0f;
            }
            for (int k = G >> 1; k > 0; k >>= 1) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], k);
                    if constexpr (GRAD) gx[u] += __shfl_xor_sync(0xffffffffu, gx[u], k);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u, o += s.oh) {
                if (h + u >= n) continue;
                const float r = rsqrtf(fmaf(sq[u], inv_d, a.eps));
                const float m = -gx[u] * r * r * inv_d;                  // -n' mean(g w n') = x r m
                const uint64_t r2 = pack2(r, r), m2 = pack2(m, m);
                R out;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    uint64_t f;
                    if constexpr (GRAD) {
                        acc[i] = fma2(g[u][i], mul2(v[u][i], r2), acc[i]);
                        f = mul2(fma2(v[u][i], m2, mul2(g[u][i], w2[i])), r2);
                    } else {
                        const uint64_t other2 = IL ? two(swapped(unpack2(v[u][i]))) : v[u][partner(i)];
                        f = mul2(fma2(other2, sn[i], mul2(v[u][i], cs[i])), r2);
                    }
                    out.set(i, unpack2(f));
                }
                out.template put<IL>(o, o + ab);
            }
        };
        // every lane of the warp takes the same turns: the sums are shuffled
        for (int h = 0; h < heads; h += 2 * U) {
            if (h + U < heads) fetch(1, h + U);
            work(0, h);
            if (h + U < heads) {
                if (h + 2 * U < heads) fetch(0, h + 2 * U);
                work(1, h + U);
            }
        }
    }

    if constexpr (GRAD) {
        if (a.part == nullptr) return;
        // sums over this block's groups in a fixed order, one row of partials a block
        const int groups = kBlock<GRAD> / G, group = threadIdx.x / G;
        if (in) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float2 f = unpack2(acc[i]);
                const int c = i < NP / 2 ? at + 2 * i : bt + 2 * i - HV;
                sm[group * a.D + c] = f.x;
                sm[group * a.D + c + 1] = f.y;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.D; i += kBlock<GRAD>) {
            float v = 0.0f;
            for (int g = 0; g < groups; ++g) v += sm[g * a.D + i];
            a.part[(int64_t)blockIdx.x * a.D + i] = v;
        }
    }
}

// Any head size, stride and alignment: a warp a row, a value a lane at a time.
template <typename T>
__device__ __forceinline__ float value(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return tok::Elem<T>::to(*p);
}
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads) k_qk_norm_rope_any(const __grid_constant__ RopeArgs a) {
    pdl_begin();
    extern __shared__ float sm[];
    constexpr int NC = kMaxD / 32;
    const int lane = threadIdx.x & 31, which = (int)blockIdx.x >= a.blocks[0];
    const Side& s = a.side[which];
    const float inv_d = 1.0f / (float)a.D;
    float acc[NC] = {};
    const int64_t rows = a.T * s.H, stride = (int64_t)a.blocks[which] * (kThreads / 32);
    for (int64_t row = (int64_t)(blockIdx.x - (which ? a.blocks[0] : 0)) * (kThreads / 32) + (threadIdx.x >> 5); row < rows; row += stride) {
        const int64_t t = row / s.H;
        const int h = (int)(row - t * s.H);
        const int64_t p = a.half ? place_of(a, t, lane == 0) * a.half : 0;
        const T* x = reinterpret_cast<const T*>(s.x) + t * s.xt + h * s.xh;
        const T* d = GRAD ? reinterpret_cast<const T*>(s.dy) + t * s.yt + h * s.yh : nullptr;
        T* o = reinterpret_cast<T*>(s.out) + t * s.ot + h * s.oh;
        float v[NC], g[NC], sq = 0.0f, gx = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = lane + 32 * c;
            v[c] = g[c] = 0.0f;
            if (i >= a.D) continue;
            v[c] = value(x + i);
            sq += v[c] * v[c];
            const bool turned = i < 2 * a.half, ahead = a.interleaved ? !(i & 1) : i < a.half;
            const int k = a.interleaved ? i / 2 : (ahead ? i : i - a.half);
            const int other = !turned ? i : (a.interleaved ? i ^ 1 : (ahead ? i + a.half : i - a.half));
            const float cs = turned ? a.cos[p + k] : 1.0f, sn = turned ? (ahead ? -a.sin[p + k] : a.sin[p + k]) : 0.0f;
            const float w = s.w ? s.w[i] : 1.0f;
            if constexpr (GRAD) {
                g[c] = value(d + i) * cs - value(d + other) * sn;
                gx += g[c] * w * v[c];
            } else {                                   // the turned row, without its norm
                g[c] = v[c] * w * cs + value(x + other) * (s.w ? s.w[other] : 1.0f) * sn;
            }
        }
        sq = warp_sum(sq);
        gx = warp_sum(gx);
        const float r = rsqrtf(fmaf(sq, inv_d, a.eps)), m = gx * r * r * inv_d;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = lane + 32 * c;
            if (i >= a.D) continue;
            float f = g[c] * r;
            if constexpr (GRAD) {
                acc[c] += g[c] * (v[c] * r);
                f = r * (g[c] * (s.w ? s.w[i] : 1.0f) - v[c] * m);
            }
            if constexpr (sizeof(T) == 4) o[i] = f;
            else o[i] = tok::Elem<T>::from(f);
        }
    }
    if constexpr (GRAD) {
        if (a.part == nullptr) return;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 32 * c < a.D) sm[(threadIdx.x >> 5) * a.D + lane + 32 * c] = acc[c];
        __syncthreads();
        for (int i = threadIdx.x; i < a.D; i += kThreads) {
            float v = 0.0f;
            for (int g = 0; g < kThreads / 32; ++g) v += sm[g * a.D + i];
            a.part[(int64_t)blockIdx.x * a.D + i] = v;
        }
    }
}

// Column sums of the partials [blocks of queries, then of keys][D]: in block order within each of 32 strands, strands in
// order.
__global__ void __launch_bounds__(1024) k_rope_weight_grad(const float* __restrict__ part, int blocks_q, int blocks_k,
                                                           int D, float* __restrict__ dqw, float* __restrict__ dkw) {
    pdl_begin();
    __shared__ float sm[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    const int b0 = blockIdx.y ? blocks_q : 0, b1 = blockIdx.y ? blocks_q + blocks_k : blocks_q;
    float v = 0.0f;
    if (col < D)
#pragma unroll 8
        for (int b = b0 + strand; b < b1; b += 32) v += part[(int64_t)b * D + col];
    sm[strand][threadIdx.x & 31] = v;
    __syncthreads();
    float* to = blockIdx.y ? dkw : dqw;
    if (strand == 0 && col < D && to) {
        float total = 0.0f;
        for (int s = 0; s < 32; ++s) total += sm[s][threadIdx.x];
        to[col] = total;
    }
}

constexpr int kMaxBlocks = kNumSMs * 8;

// Blocks of each side.  Forwards every warp has one item.  Backwards a block leaves a row of partial sums, so there are at
// most about kMaxBlocks, shared in proportion to the sides' rows, and every warp of a side has the same number of items.
void share_blocks(RopeArgs& a, const int64_t (&want)[2], bool grad) {
    const int64_t rows = (int64_t)a.side[0].H + a.side[1].H;
    for (int i = 0; i < 2; ++i) {
        const int64_t most = grad ? std::max<int64_t>(1, (int64_t)kMaxBlocks * a.side[i].H / rows) : (int64_t)1 << 30;
        const int64_t each = std::max<int64_t>(1, (want[i] + most - 1) / most);
        a.blocks[i] = (int)((want[i] + each - 1) / each);
    }
}

template <typename T, int V, bool GRAD>
int plan(RopeArgs& a, cudaStream_t s) {
    int G = 1;
    while (G * V < a.D) G *= 2;
    // Heads per item: a token's angles are reused over an item's heads, but a small batch needs the items.  All heads
    // while that leaves 16 warps a SM, else one.
    const bool wide = a.T * G >= (int64_t)kNumSMs * 512;
    const int64_t per_block = (int64_t)(kBlock<GRAD> / 32) * (32 / G);
    int64_t want[2];
    for (int i = 0; i < 2; ++i) {
        a.heads[i] = wide ? a.side[i].H : 1;
        a.chunks[i] = wide ? a.side[i].H > 0 : a.side[i].H;
        want[i] = (a.T * a.chunks[i] + per_block - 1) / per_block;
    }
    share_blocks(a, want, GRAD);
    const size_t smem = GRAD ? (size_t)(kBlock<GRAD> / G) * a.D * sizeof(float) : 0;
    const int blocks = a.blocks[0] + a.blocks[1];
    constexpr int U = 2;
    if (a.interleaved) k_qk_norm_rope<T, V, U, GRAD, true><<<blocks, kBlock<GRAD>, smem, s>>>(a, G);
    else k_qk_norm_rope<T, V, U, GRAD, false><<<blocks, kBlock<GRAD>, smem, s>>>(a, G);
    PMG_LAUNCH_CHECK();
    return PMG_OK;
}

template <typename T, bool GRAD>
int plan_any(RopeArgs& a, cudaStream_t s) {
    int64_t want[2];
    for (int i = 0; i < 2; ++i) want[i] = (a.T * a.side[i].H + kThreads / 32 - 1) / (kThreads / 32);
    share_blocks(a, want, GRAD);
    const size_t smem = GRAD ? (size_t)(kThreads / 32) * a.D * sizeof(float) : 0;
    k_qk_norm_rope_any<T, GRAD><<<a.blocks[0] + a.blocks[1], kThreads, smem, s>>>(a);
    PMG_LAUNCH_CHECK();
    return PMG_OK;
}

// Whether a lane's V values can be read as one vector (interleaved) or two, and the angles as pairs.
bool aligned(const RopeArgs& a, int V, int size, bool grad) {
    const int unit = a.interleaved ? V : V / 2;
    auto ok = [&](const void* p, int64_t t, int64_t h) {
        return ((uintptr_t)p % (unit * size)) == 0 && t % unit == 0 && h % unit == 0;
    };
    for (const Side& s : a.side) {
        if (s.H == 0) continue;
        if (!ok(s.x, s.xt, s.xh) || !ok(s.out, s.ot, s.oh) || (grad && !ok(s.dy, s.yt, s.yh))) return false;
    }
    if (((uintptr_t)a.cos | (uintptr_t)a.sin) & 7) return false;
    return a.D % V == 0 && a.D <= 32 * V && (2 * a.half) % V == 0 && a.half % 2 == 0;
}

template <typename T, bool GRAD>
int by_width(RopeArgs& a, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (aligned(a, W, sizeof(T), GRAD)) return plan<T, W, GRAD>(a, s);
    if constexpr (sizeof(T) == 2) {
        if (aligned(a, 4, 2, GRAD)) return plan<T, 4, GRAD>(a, s);
    }
    return plan_any<T, GRAD>(a, s);
}

template <bool GRAD>
int by_type(int dtype, RopeArgs& a, cudaStream_t s) {
    switch (dtype) {
        case PMG_BF16: return by_width<__nv_bfloat16, GRAD>(a, s);
        case PMG_F16: return by_width<__half, GRAD>(a, s);
        default: return by_width<float, GRAD>(a, s);
    }
}

int check(int dtype, int64_t T, int Hq, int Hk, int D, int rot, int places, const float* cos, const float* sin) {
    if (dtype != PMG_F32 && dtype != PMG_F16 && dtype != PMG_BF16) return PMG_ERR_UNSUPPORTED;
    if (T < 0 || Hq < 0 || Hk < 0 || D < 1 || rot < 0 || (rot & 1) || rot > D) return PMG_ERR_BAD_ARG;
    if (rot > 0 && (!cos || !sin || places < 1)) return PMG_ERR_BAD_ARG;
    if (D > kMaxD || T > (int64_t)1 << 31 || Hq > 4096 || Hk > 4096) return PMG_ERR_UNSUPPORTED;
    return PMG_OK;
}

}  // namespace
}  // namespace pmg

using namespace pmg;

extern "C" int pmg_qk_norm_rope(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok,
                                int64_t k_head, int32_t dtype, int64_t T, int32_t Hq, int32_t Hk, int32_t D,
                                int32_t rot, const float* q_weight, const float* k_weight, const float* cos,
                                const float* sin, int32_t places, const int32_t* positions, float eps,
                                int32_t interleaved, void* q_out, int64_t qo_tok, int64_t qo_head, void* k_out,
                                int64_t ko_tok, int64_t ko_head, int32_t* status, void* stream) {
    const int rc = check(dtype, T, Hq, Hk, D, rot, places, cos, sin);
    if (rc != PMG_OK) return rc;
    if (T == 0 || Hq + Hk == 0) return PMG_OK;
    if ((Hq && (!q || !q_out)) || (Hk && (!k || !k_out))) return PMG_ERR_BAD_ARG;
    RopeArgs a{};
    a.side[0] = {q, nullptr, q_out, q_weight, q_tok, q_head, 0, 0, qo_tok, qo_head, Hq};
    a.side[1] = {k, nullptr, k_out, k_weight, k_tok, k_head, 0, 0, ko_tok, ko_head, Hk};
    a.cos = cos; a.sin = sin; a.pos = rot ? positions : nullptr; a.T = T; a.places = rot ? places : INT32_MAX; a.D = D;
    a.half = rot / 2; a.interleaved = interleaved != 0; a.eps = eps; a.status = status;
    return by_type<false>(dtype, a, as_stream(stream));
}

extern "C" size_t pmg_qk_norm_rope_grad_workspace_bytes(int32_t D) {
    return (size_t)(kMaxBlocks + 2) * (D > 0 ? D : 0) * sizeof(float);
}

extern "C" int pmg_qk_norm_rope_grad(const void* dq, int64_t dq_tok, int64_t dq_head, const void* dk, int64_t dk_tok,
                                     int64_t dk_head, const void* q, int64_t q_tok, int64_t q_head, const void* k,
                                     int64_t k_tok, int64_t k_head, int32_t dtype, int64_t T, int32_t Hq, int32_t Hk,
                                     int32_t D, int32_t rot, const float* q_weight, const float* k_weight,
                                     const float* cos, const float* sin, int32_t places, const int32_t* positions,
                                     float eps, int32_t interleaved, void* q_grad, int64_t qo_tok, int64_t qo_head,
                                     void* k_grad, int64_t ko_tok, int64_t ko_head, float* q_weight_grad,
                                     float* k_weight_grad, void* workspace, size_t workspace_bytes, int32_t* status,
                                     void* stream) {
    const int rc = check(dtype, T, Hq, Hk, D, rot, places, cos, sin);
    if (rc != PMG_OK) return rc;
    cudaStream_t s = as_stream(stream);
    const bool weights = q_weight_grad || k_weight_grad;
    if (T == 0 || Hq + Hk == 0) {
        if (q_weight_grad) PMG_CUDA_TRY(cudaMemsetAsync(q_weight_grad, 0, D * sizeof(float), s));
        if (k_weight_grad) PMG_CUDA_TRY(cudaMemsetAsync(k_weight_grad, 0, D * sizeof(float), s));
        return PMG_OK;
    }
    if ((Hq && (!q || !dq || !q_grad)) || (Hk && (!k || !dk || !k_grad))) return PMG_ERR_BAD_ARG;
    if (weights && (!workspace || workspace_bytes < pmg_qk_norm_rope_grad_workspace_bytes(D))) return PMG_ERR_BAD_ARG;
    RopeArgs a{};
    a.side[0] = {q, dq, q_grad, q_weight, q_tok, q_head, dq_tok, dq_head, qo_tok, qo_head, Hq};
    a.side[1] = {k, dk, k_grad, k_weight, k_tok, k_head, dk_tok, dk_head, ko_tok, ko_head, Hk};
    a.cos = cos; a.sin = sin; a.pos = rot ? positions : nullptr; a.T = T; a.places = rot ? places : INT32_MAX; a.D = D;
    a.half = rot / 2; a.interleaved = interleaved != 0; a.eps = eps; a.status = status;
    a.part = weights ? static_cast<float*>(workspace) : nullptr;
    const int rc2 = by_type<true>(dtype, a, s);
    if (rc2 != PMG_OK) return rc2;
    if (weights) {
        return launch_after(k_rope_weight_grad, dim3((D + 31) / 32, 2), 1024, 0, s, (const float*)a.part, a.blocks[0],
                            a.blocks[1], D, q_weight_grad, k_weight_grad);
    }
    return PMG_OK;
}
