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
// row (D values as 16-byte vectors, one a lane) and walks several heads of one token with that token's angles in
// registers: the angles are 8 bytes per pair against 2 bytes per value, so loading them per head would cost more
// first-level cache traffic than the heads themselves.  The partner of a value in the other half of the head is loaded
// again (a first-level hit) rather than shuffled: one load against one shuffle per two values.
// Sums and norms are fp32; a value is rounded once, when it is stored.
#include <algorithm>

#include "tok_common.cuh"

namespace pmg {
namespace {

constexpr int kThreads = 256;
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
    int places, D, half, interleaved, heads, chunks[2];   // heads per item; items per token of each side
    float eps;
    int32_t* status;
    float* part;              // gradients of w: [blocks][2][D]
};

template <typename T, int V> struct Vec;
template <int V> struct alignas(2 * V) Raw16 { uint16_t v[V]; };
template <int V> struct alignas(4 * V) Raw32 { float v[V]; };
template <int V> struct Vec<__half, V> { using type = Raw16<V>; };
template <int V> struct Vec<__nv_bfloat16, V> { using type = Raw16<V>; };
template <int V> struct Vec<float, V> { using type = Raw32<V>; };

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V]) {
    typename Vec<T, V>::type r = *reinterpret_cast<const typename Vec<T, V>::type*>(p);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = r.v[i];
    } else {
        const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = tok::Elem<T>::to(t[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
    typename Vec<T, V>::type r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = f[i];
    } else {
        T* t = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = tok::Elem<T>::from(f[i]);
    }
    *reinterpret_cast<typename Vec<T, V>::type*>(p) = r;
}

// G lanes per row; NCH vectors of V values a lane; U heads at once.
template <typename T, int V, int NCH, int U, bool GRAD>
__global__ void __launch_bounds__(kThreads) k_qk_norm_rope(const __grid_constant__ RopeArgs a, int G) {
    pdl_begin();
    extern __shared__ float sm[];
    const int lane = threadIdx.x & 31, per_warp = 32 / G, gi = lane / G, gl = lane % G;
    const int64_t per_token = a.chunks[0] + a.chunks[1], items = a.T * per_token;
    const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int64_t stride = (int64_t)gridDim.x * (kThreads / 32) * per_warp;
    const float inv_d = 1.0f / (float)a.D;
    const int rot = 2 * a.half;
    float acc[GRAD ? 2 : 1][NCH][V];
    if constexpr (GRAD) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[s][c][e] = 0.0f;
    }

    for (int64_t base = warp * per_warp; base < items; base += stride) {
        const bool live = base + gi < items;
        const int64_t item = live ? base + gi : items - 1;
        const int64_t t = item / per_token;
        int chunk = (int)(item - t * per_token);
        const int which = chunk >= a.chunks[0];
        if (which) chunk -= a.chunks[0];
        const Side& s = a.side[which];
        const int h0 = chunk * a.heads, h1 = live ? min(h0 + a.heads, s.H) : h0;
        int p = a.pos ? a.pos[t] : (int)t;
        if (p < 0 || p >= a.places) {
            if (live && gl == 0) flag(a.status, PMG_ERR_RANGE);
            p = 0;
        }
        // own and partner places, angles (sign folded into sn) and weights of this lane's vectors
        float cs[NCH][V], sn[NCH][V], w[NCH][V], wp[NCH][V];
        int at[NCH], other[NCH];
        bool in[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int i0 = (gl + c * G) * V;
            in[c] = i0 < a.D;
            at[c] = in[c] ? i0 : 0;
            other[c] = at[c];
            const bool turned = at[c] < rot;
            const bool first = at[c] < a.half;
            if (turned && !a.interleaved) other[c] = first ? at[c] + a.half : at[c] - a.half;
            if (V == 1 && turned && a.interleaved) other[c] = at[c] ^ 1;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = at[c] + e;
                cs[c][e] = 1.0f;
                sn[c][e] = 0.0f;
                if (turned) {
                    const int k = a.interleaved ? i >> 1 : (first ? i : i - a.half);
                    const bool neg = a.interleaved ? !(i & 1) : first;
                    cs[c][e] = a.cos[(int64_t)p * a.half + k];
                    const float v = a.sin[(int64_t)p * a.half + k];
                    sn[c][e] = neg ? -v : v;
                }
                w[c][e] = s.w ? s.w[i] : 1.0f;
            }
            if constexpr (!GRAD) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int i = (V > 1 && a.interleaved) ? at[c] + (e ^ 1) : other[c] + e;
                    wp[c][e] = s.w ? s.w[i] : 1.0f;
                }
            }
        }
        const T* xt = reinterpret_cast<const T*>(s.x) + t * s.xt;
        const T* yt = GRAD ? reinterpret_cast<const T*>(s.dy) + t * s.yt : nullptr;
        T* ot = reinterpret_cast<T*>(s.out) + t * s.ot;
        const bool swap = V > 1 && a.interleaved;
        for (int hb = 0; hb < a.heads; hb += U) {
            float x[U][NCH][V], y[U][NCH][V];   // x; its partner (forwards) or g (backwards)
            float sq[U], gx[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + hb + u;
                const bool on = h < h1;
                sq[u] = gx[u] = 0.0f;
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    float d[V], dp[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) x[u][c][e] = y[u][c][e] = d[e] = dp[e] = 0.0f;
                    if (on && in[c]) {
                        load<T, V>(xt + h * s.xh + at[c], x[u][c]);
                        const T* src = GRAD ? yt + h * s.yh : xt + h * s.xh;
                        if constexpr (GRAD) load<T, V>(src + at[c], d);
                        if (!swap) load<T, V>(src + other[c], dp);
                    }
                    if (swap) {
#pragma unroll
                        for (int e = 0; e < V; ++e) dp[e] = GRAD ? d[e ^ (V > 1)] : x[u][c][e ^ (V > 1)];
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        y[u][c][e] = GRAD ? d[e] * cs[c][e] - dp[e] * sn[c][e] : dp[e];
                        sq[u] += x[u][c][e] * x[u][c][e];
                        if constexpr (GRAD) gx[u] += y[u][c][e] * w[c][e] * x[u][c][e];
                    }
                }
            }
            for (int o = G >> 1; o > 0; o >>= 1) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], o);
                    if constexpr (GRAD) gx[u] += __shfl_xor_sync(0xffffffffu, gx[u], o);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + hb + u;
                const float r = rsqrtf(sq[u] * inv_d + a.eps);
                const float m = GRAD ? gx[u] * r * r * inv_d : 0.0f;   // n' mean(g w n') = x r m'
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        if constexpr (GRAD) {
                            if (which) acc[1][c][e] += y[u][c][e] * (x[u][c][e] * r);
                            else acc[0][c][e] += y[u][c][e] * (x[u][c][e] * r);
                            o[e] = r * (y[u][c][e] * w[c][e] - x[u][c][e] * m);
                        } else {
                            o[e] = (x[u][c][e] * r * w[c][e]) * cs[c][e] + (y[u][c][e] * r * wp[c][e]) * sn[c][e];
                        }
                    }
                    if (h < h1 && in[c]) store<T, V>(ot + h * s.oh + at[c], o);
                }
            }
        }
    }

    if constexpr (GRAD) {
        if (a.part == nullptr) return;
        // sums over this block's groups in a fixed order, one row of partials a block
        const int groups = kThreads / G, group = threadIdx.x / G;
        for (int s = 0; s < 2; ++s) {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int i = (gl + c * G) * V + e;
                    if (i < a.D) sm[group * a.D + i] = s ? acc[GRAD ? 1 : 0][c][e] : acc[0][c][e];
                }
            __syncthreads();
            for (int i = threadIdx.x; i < a.D; i += kThreads) {
                float v = 0.0f;
                for (int g = 0; g < groups; ++g) v += sm[g * a.D + i];
                a.part[((int64_t)blockIdx.x * 2 + s) * a.D + i] = v;
            }
        }
    }
}

// Column sums of the partials [blocks][2][D] in block order within each of 32 strands, strands in order.
__global__ void __launch_bounds__(1024) k_rope_weight_grad(const float* __restrict__ part, int blocks, int D,
                                                           float* __restrict__ dqw, float* __restrict__ dkw) {
    pdl_begin();
    __shared__ float sm[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5, width = 2 * D;
    float v = 0.0f;
    if (col < width)
        for (int b = strand; b < blocks; b += 32) v += part[(int64_t)b * width + col];
    sm[strand][threadIdx.x & 31] = v;
    __syncthreads();
    if (strand == 0 && col < width) {
        float total = 0.0f;
        for (int s = 0; s < 32; ++s) total += sm[s][threadIdx.x];
        float* to = col < D ? dqw : dkw;
        if (to) to[col < D ? col : col - D] = total;
    }
}

constexpr int kMaxBlocks = kNumSMs * 4;

template <typename T, int V, int NCH, int U, bool GRAD>
int launch(const RopeArgs& a, int G, int blocks, cudaStream_t s) {
    const size_t smem = GRAD ? (size_t)(kThreads / G) * a.D * sizeof(float) : 0;
    k_qk_norm_rope<T, V, NCH, U, GRAD><<<blocks, kThreads, smem, s>>>(a, G);
    PMG_LAUNCH_CHECK();
    return PMG_OK;
}

template <typename T, int V, int NCH, bool GRAD>
int plan(RopeArgs& a, float* part, int* blocks_out, cudaStream_t s) {
    int G = 1;
    while (G < 32 && G * V < a.D) G *= 2;
    // Heads per item: all of a token's angles are reused over an item's heads, but a small batch needs the items.
    // Four at once while that leaves 16 warps a SM; measured figures beside the entry points below.
    const int64_t groups4 = a.T * ((a.side[0].H + 3) / 4 + (a.side[1].H + 3) / 4);
    const bool wide = groups4 * G >= (int64_t)kNumSMs * 512;
    a.heads = wide ? 4 : 1;
    int64_t items = 0;
    for (int i = 0; i < 2; ++i) {
        a.chunks[i] = (a.side[i].H + a.heads - 1) / a.heads;
        items += a.T * a.chunks[i];
    }
    const int64_t per_block = (int64_t)(kThreads / 32) * (32 / G);
    int64_t blocks = std::max<int64_t>(1, (items + per_block - 1) / per_block);
    if (GRAD) blocks = std::min<int64_t>(blocks, kMaxBlocks);
    else blocks = std::min<int64_t>(blocks, (int64_t)1 << 20);
    *blocks_out = (int)blocks;
    a.part = part;
    return wide ? launch<T, V, NCH, (NCH * V > 8 ? 2 : 4), GRAD>(a, G, (int)blocks, s)
                : launch<T, V, NCH, 1, GRAD>(a, G, (int)blocks, s);
}

bool aligned(const RopeArgs& a, int V, int size, bool grad) {
    auto ok = [&](const void* p, int64_t t, int64_t h) {
        return ((uintptr_t)p % (V * size)) == 0 && t % V == 0 && h % V == 0;
    };
    for (const Side& s : a.side) {
        if (s.H == 0) continue;
        if (!ok(s.x, s.xt, s.xh) || !ok(s.out, s.ot, s.oh) || (grad && !ok(s.dy, s.yt, s.yh))) return false;
    }
    return a.D % V == 0 && (a.interleaved ? (2 * a.half) % V == 0 : a.half % V == 0);
}

template <typename T, bool GRAD>
int by_width(RopeArgs& a, float* part, int* blocks, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (aligned(a, W, sizeof(T), GRAD))
        return a.D <= 32 * W ? plan<T, W, 1, GRAD>(a, part, blocks, s) : plan<T, W, 2, GRAD>(a, part, blocks, s);
    if constexpr (sizeof(T) == 2) {
        if (aligned(a, 4, 2, GRAD)) return plan<T, 4, 2, GRAD>(a, part, blocks, s);
    }
    return plan<T, 1, 8, GRAD>(a, part, blocks, s);
}

template <bool GRAD>
int by_type(int dtype, RopeArgs& a, float* part, int* blocks, cudaStream_t s) {
    switch (dtype) {
        case PMG_BF16: return by_width<__nv_bfloat16, GRAD>(a, part, blocks, s);
        case PMG_F16: return by_width<__half, GRAD>(a, part, blocks, s);
        default: return by_width<float, GRAD>(a, part, blocks, s);
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
    a.cos = cos; a.sin = sin; a.pos = positions; a.T = T; a.places = rot ? places : INT32_MAX; a.D = D;
    a.half = rot / 2; a.interleaved = interleaved != 0; a.eps = eps; a.status = status;
    int blocks = 0;
    return by_type<false>(dtype, a, nullptr, &blocks, as_stream(stream));
}

extern "C" size_t pmg_qk_norm_rope_grad_workspace_bytes(int32_t D) {
    return (size_t)kMaxBlocks * 2 * (D > 0 ? D : 0) * sizeof(float);
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
    a.cos = cos; a.sin = sin; a.pos = positions; a.T = T; a.places = rot ? places : INT32_MAX; a.D = D;
    a.half = rot / 2; a.interleaved = interleaved != 0; a.eps = eps; a.status = status;
    int blocks = 0;
    const int rc2 = by_type<true>(dtype, a, weights ? static_cast<float*>(workspace) : nullptr, &blocks, s);
    if (rc2 != PMG_OK) return rc2;
    if (weights) {
        k_rope_weight_grad<<<(2 * D + 31) / 32, 1024, 0, s>>>(static_cast<const float*>(workspace), blocks, D,
                                                              q_weight_grad, k_weight_grad);
        PMG_LAUNCH_CHECK();
    }
    return PMG_OK;
}
