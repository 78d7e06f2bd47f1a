// Linear layer with everything behind the product fused into its epilogue, and its gradients.
//
//   z = x W^T + b,   y = act(z) + r          x [M, K], W [N, K], r and y [M, N]; act: none, relu, silu, gelu (erf)
//   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz     (dr is dy itself)
//
// Three kernels do the products.
//   k_rows    up to 32 rows: bound by one read of W.  A block owns 16 output columns, its warps split K; mma.sync with W
//             as the 16-row operand, every lane's 16-byte load feeding two instructions (a dot product does not mind the
//             order of K, so no shuffle or shared-memory transpose is needed).
//   k_gemm    everything larger: tcgen05 with tiles of 128 x 64, 128 x 128 or, by pairs of CTAs, 256 x 256, TMA ring,
//             accumulators double-buffered in tensor memory so that the epilogue of one tile runs under the next one's
//             products; sixteen warps take it, straight from registers to memory.
//   k_split_sum   the last wave of tiles, when it would leave most SMs idle, is cut along K into fp32 partials that this
//             kernel adds in split order (no atomics: results do not depend on timing) and takes through the epilogue.
// Measured: 38,400 x 1024 x 4096 with gelu 252 us (1280 TFLOP/s) alone and 295 to 310 in long runs, where the power limit holds
// the clock at 1.1 to 1.3 GHz (without the activation 271 to 283; cuBLAS 279); its gradients over 9600 rows 164 us, 1200 x 1024
// x 1024 10 us, one row 1024 -> 4096 3.5 us (2.4 TB/s).  With eight warps that staged their rows in shared memory the first took
// 278 us, and 321 in long runs.
// dz is rounded to the operands' 16-bit type before its two products (tensor cores take no other), db is summed from the
// unrounded fp32 values.
#include <algorithm>

#include "tok_common.cuh"

namespace pmg {
namespace {

using namespace tok;

// ----------------------------------------------------------------------------------------------------------------- //
// Activations
// ----------------------------------------------------------------------------------------------------------------- //

// gelu(x) = x Phi(x) = max(x, 0) - a Phi(-a), a = |x|, with its limit 0 at -inf: what is approximated is the tail Phi(-a), and
// its relative error is that of a negative result.  Behind a = 13 Phi(-a) is under 2^-126 and comes out as 0.
//
// For 16-bit results Phi(-a) = 2^q(a): q is smooth, so a short polynomial holds it (least largest weighted error, by linear
// programming on a grid).  fp16, which turns to 0 at 5.8: degree 6, relative error of Phi 4.2e-5 (2^-14; the type rounds to
// 2^-11).  bf16: degree 8, 2.4e-4 up to 13 (2^-12; the type rounds to 2^-8).  Both evaluated in fp32.  A product whose tiles
// keep the tensor cores busy runs at the power limit, where each operation per output counts as energy: 10 or 11 of them,
// in place of the 20 of the finer form.
template <typename T> struct Tail;
template <> struct Tail<__half> {
    static constexpr int kDegree = 6;
    static __device__ __forceinline__ constexpr float at(int i) {
        constexpr float c[] = {-1.000057179e+00f, -1.150326502e+00f, -4.609019817e-01f, -5.148804179e-02f, 7.304450847e-03f,
                               -6.289135209e-04f, 2.407393613e-05f};
        return c[i];
    }
};
template <> struct Tail<__nv_bfloat16> {
    static constexpr int kDegree = 8;
    static __device__ __forceinline__ constexpr float at(int i) {
        constexpr float c[] = {-1.000191180e+00f, -1.150026044e+00f, -4.608018950e-01f, -5.209471939e-02f, 7.814329701e-03f,
                               -8.084457054e-04f, 5.337338495e-05f, -2.002034972e-06f, 3.226851094e-08f};
        return c[i];
    }
};

// For fp32 results, and for the slope: Phi(-a) = 2^(-a^2 / 2 log2 e) t P(t), t = 1 / (1 + 0.3 a) (least squares, repeated with
// weights times the error).  P of degree 7 with least largest relative error, 1.2e-7, 5e-7 in fp32.  The slope's, of degree
// 5, has least largest error relative to t P(t) + a / sqrt(2 pi), the size of what it is added to: 6e-7.
__device__ constexpr float kMills[8] = {1.196245409e-01f, 1.208263142e-01f, 9.946506889e-02f, 1.300325943e-01f,
                                        -5.645003673e-02f, 2.093463112e-01f, -1.589336760e-01f, 3.608882384e-02f};
__device__ constexpr float kSlope[6] = {1.200557486e-01f, 1.135166463e-01f, 1.463589779e-01f, -2.274043795e-02f,
                                        2.222955805e-01f, -7.948681410e-02f};
constexpr float kHalfLog2e = 0.72134752f, kHalfLog2eRest = (float)(0.72134752044448170368 - (double)kHalfLog2e);
// One value at a time: constants of packed operations take registers, which the epilogue does not have.
__device__ __forceinline__ float gelu_fine(float a) {
    const float x = fminf(fabsf(a), 14.0f), t = rcp_approx(fmaf(x, 0.3f, 1.0f));
    float p = kMills[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = fmaf(p, t, kMills[i]);
    const float sq = x * x, y = sq * -kHalfLog2e;
    // what rounding the exponent loses (up to 2^-17 of the result): k sq - y, k (x^2 - sq), and the rest of k
    float r = fmaf(sq, -kHalfLog2e, -y);
    r = fmaf(fmaf(x, x, -sq), -kHalfLog2e, r);
    r = fmaf(sq, -kHalfLog2eRest, r);
    const float e = ex2(y);
    return fmaf(-x, p * t * fmaf(e * kLn2, r, e), max_nan(a, 0.0f));
}
template <typename T>
__device__ __forceinline__ void gelu_pair(float& a, float& b) {
    const float xa = fminf(fabsf(a), 14.0f), xb = fminf(fabsf(b), 14.0f);
    const uint64_t x = pack2(xa, xb);
    constexpr int N = Tail<T>::kDegree;
    uint64_t p = pack2(Tail<T>::at(N), Tail<T>::at(N));
#pragma unroll
    for (int i = N - 1; i >= 0; --i) p = fma2(p, x, pack2(Tail<T>::at(i), Tail<T>::at(i)));
    const float2 f = unpack2(ex2_pair(p));               // Phi(-|x|)
    a = fmaf(-xa, f.x, max_nan(a, 0.0f));
    b = fmaf(-xb, f.y, max_nan(b, 0.0f));
}

// N values, the choice made once for all of them; fine: for an fp32 result.
template <typename T, int N>
__device__ __forceinline__ void activate(int act, bool fine, float* v) {
    if (act == PMG_ACT_GELU && fine) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gelu_fine(v[i]);
    } else if (act == PMG_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; i += 2) gelu_pair<T>(v[i], v[i + 1]);
    } else if (act == PMG_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= rcp_approx(1.0f + ex2(-v[i] * kLog2e));
    } else if (act == PMG_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = max_nan(v[i], 0.0f);
    }
}

// dz = dy act'(z) for 8 values.  gelu' = Phi(z) + z phi(z) is G(a) = 2^(-a^2 / 2 log2 e) (t P(t) - a / sqrt(2 pi)) for z = -a and
// 1 - G(a) for z = a.  With erff and expf this pass took 75 us for 9600 x 4096, four fifths of it arithmetic; now 50 (4.7 TB/s).
__device__ __forceinline__ void times_slope(int act, float (&g)[8], const float (&z)[8]) {
    if (act == PMG_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {                    // one by one: constants of packed operations take registers
            const float x = fabsf(z[i]), t = rcp_approx(fmaf(x, 0.3f, 1.0f));
            float p = kSlope[5];
#pragma unroll
            for (int k = 4; k >= 0; --k) p = fmaf(p, t, kSlope[k]);
            const float f = fmaf(p, t, x * -0.39894228f) * ex2(x * x * -kHalfLog2e);
            g[i] *= z[i] < 0.0f ? f : 1.0f - f;
        }
    } else if (act == PMG_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = rcp_approx(1.0f + ex2(-z[i] * kLog2e));
            g[i] *= s * fmaf(z[i], 1.0f - s, 1.0f);
        }
    } else if (act == PMG_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = z[i] > 0.0f ? g[i] : 0.0f;
    }
}

// ----------------------------------------------------------------------------------------------------------------- //
// The epilogue's destination
// ----------------------------------------------------------------------------------------------------------------- //
struct Out {
    const void* bias;        // [N] of the operands' type, or null
    const void* resid;       // [M, N] of y's type, or null
    void* y;
    void* pre;               // z of the operands' type, or null
    int64_t ldr, ldy, ldp;
    int act;
    int f32;                 // y and the residual are fp32, else the operands' type
    int vec;                 // rows of y, resid and pre start on boundaries of 16 bytes (1), 32 (2) or less (0)
};

// 8 values z[0..7] of row m from column n on: bias, activation, residual, stores.  Used where rows are not staged.
template <typename T>
__device__ __forceinline__ void finish8(const Out& o, int64_t m, int n, int N, float (&z)[8]) {
    const int cnt = min(8, N - n);
    if (o.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < cnt) z[i] += Elem<T>::to(static_cast<const T*>(o.bias)[n + i]);
    }
    const bool vec = o.vec && cnt == 8;
    if (o.pre) {
        T* p = static_cast<T*>(o.pre) + m * o.ldp + n;
        if (vec) {
            *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::pack(z[0], z[1]), Elem<T>::pack(z[2], z[3]),
                                                      Elem<T>::pack(z[4], z[5]), Elem<T>::pack(z[6], z[7]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < cnt) p[i] = Elem<T>::from(z[i]);
        }
    }
    activate<T, 8>(o.act, o.f32, z);
    if (o.f32) {
        if (o.resid) {
            const float* r = static_cast<const float*>(o.resid) + m * o.ldr + n;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < cnt) z[i] += r[i];
        }
        float* p = static_cast<float*>(o.y) + m * o.ldy + n;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < cnt) p[i] = z[i];
        return;
    }
    if (o.resid) {
        const T* r = static_cast<const T*>(o.resid) + m * o.ldr + n;
        if (vec) {
            const uint4 v = *reinterpret_cast<const uint4*>(r);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = Elem<T>::unpack(w[i]);
                z[2 * i] += f.x;
                z[2 * i + 1] += f.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < cnt) z[i] += Elem<T>::to(r[i]);
        }
    }
    T* p = static_cast<T*>(o.y) + m * o.ldy + n;
    if (vec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(Elem<T>::pack(z[0], z[1]), Elem<T>::pack(z[2], z[3]),
                                                  Elem<T>::pack(z[4], z[5]), Elem<T>::pack(z[6], z[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < cnt) p[i] = Elem<T>::from(z[i]);
    }
}

// ----------------------------------------------------------------------------------------------------------------- //
// Few rows
// ----------------------------------------------------------------------------------------------------------------- //
template <typename T>
__device__ __forceinline__ void mma_16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    if constexpr (Elem<T>::kFmt == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 values of a row from column k on, zero beyond K or for an absent row.
template <bool ALIGNED>
__device__ __forceinline__ uint4 row8(const uint16_t* row, int k, int K, bool on) {
    if constexpr (ALIGNED) {
        return on && k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (on && k + i < K) w[i >> 1] |= (uint32_t)row[k + i] << (16 * (i & 1));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

constexpr int kRowsCols = 16;

// NT groups of 8 rows; ALIGNED: K % 8 == 0 and rows on 16-byte boundaries.
template <typename T, int NT, bool ALIGNED>
__global__ void __launch_bounds__(512) k_rows(const uint16_t* __restrict__ x, int64_t ldx,
                                              const uint16_t* __restrict__ w, int64_t ldw, int M, int N, int K, Out o) {
    pdl_begin();
    extern __shared__ float part[];                  // [warps][16 columns][8 NT rows]
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;
    const int n0 = blockIdx.x * kRowsCols;
    const uint16_t* w0 = w + (int64_t)(n0 + g) * ldw;
    const uint16_t* w1 = w0 + 8 * ldw;
    const bool on0 = n0 + g < N, on1 = n0 + g + 8 < N;
    float acc[NT][4] = {};
    constexpr int U = NT <= 2 ? 4 : 2;
    for (int k0 = warp * 32; k0 < K; k0 += warps * 32 * U) {
        uint4 a[U], b[U], v[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * warps * 32 + 8 * q;
            a[u] = row8<ALIGNED>(w0, k, K, on0);
            b[u] = row8<ALIGNED>(w1, k, K, on1);
#pragma unroll
            for (int t = 0; t < NT; ++t) v[u][t] = row8<ALIGNED>(x + (int64_t)(8 * t + g) * ldx, k, K, 8 * t + g < M);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma_16n8k16<T>(acc[t], a[u].x, b[u].x, a[u].y, b[u].y, v[u][t].x, v[u][t].y);
                mma_16n8k16<T>(acc[t], a[u].z, b[u].z, a[u].w, b[u].w, v[u][t].z, v[u][t].w);
            }
    }
    float* mine = part + warp * (kRowsCols * 8 * NT);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int m = 8 * t + 2 * q;
        mine[m * kRowsCols + g] = acc[t][0];
        mine[(m + 1) * kRowsCols + g] = acc[t][1];
        mine[m * kRowsCols + g + 8] = acc[t][2];
        mine[(m + 1) * kRowsCols + g + 8] = acc[t][3];
    }
    __syncthreads();
    // one thread per row and pair of columns
    for (int i = threadIdx.x; i < 8 * NT * (kRowsCols / 2); i += blockDim.x) {
        const int m = i / (kRowsCols / 2), c = (i % (kRowsCols / 2)) * 2, n = n0 + c;
        if (m >= M || n >= N) continue;
        float z[2] = {0.0f, 0.0f};
        for (int s = 0; s < warps; ++s) {
            const float2 p = *reinterpret_cast<const float2*>(part + s * (kRowsCols * 8 * NT) + m * kRowsCols + c);
            z[0] += p.x;
            z[1] += p.y;
        }
        const bool two = n + 1 < N;
        if (o.bias) {
            z[0] += Elem<T>::to(static_cast<const T*>(o.bias)[n]);
            if (two) z[1] += Elem<T>::to(static_cast<const T*>(o.bias)[n + 1]);
        }
        if (o.pre) {
            T* p = static_cast<T*>(o.pre) + m * o.ldp + n;
            p[0] = Elem<T>::from(z[0]);
            if (two) p[1] = Elem<T>::from(z[1]);
        }
        activate<T, 2>(o.act, o.f32, z);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (e && !two) break;
            float v = z[e];
            if (o.f32) {
                if (o.resid) v += static_cast<const float*>(o.resid)[m * o.ldr + n + e];
                static_cast<float*>(o.y)[m * o.ldy + n + e] = v;
            } else {
                if (o.resid) v += Elem<T>::to(static_cast<const T*>(o.resid)[m * o.ldr + n + e]);
                static_cast<T*>(o.y)[m * o.ldy + n + e] = Elem<T>::from(v);
            }
        }
    }
}

// ----------------------------------------------------------------------------------------------------------------- //
// Tiles
// ----------------------------------------------------------------------------------------------------------------- //
constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 16, kFirstEpi = 4;
constexpr int kGemmThreads = 32 * (kFirstEpi + kEpiWarps);

template <int BN>
struct Cfg {
    // 256 columns: two CTAs on a tile of 256 rows, half the columns' operand in each.  A SM then loads 32 KB for what takes
    // 48 KB alone; under the power limit, which long runs meet, that is worth more than where the loads keep up.
    static constexpr bool kPair = BN == 256;
    static constexpr int kRows = kPair ? 2 * kBM : kBM, kOwnN = kPair ? BN / 2 : BN;
    static constexpr int kA = kBM * kBK * 2, kB = kOwnN * kBK * 2, kStage = kA + kB;
    static constexpr int kStages = 196608 / kStage > 8 ? 8 : 196608 / kStage;
    static constexpr int kBias = 4 * BN * 2;                   // a quarter of the columns a warp, in the operands' type
    static constexpr int kBars = kStages * kStage + kBias;
    static constexpr int kSmem = kBars + 256;
};

// What a CTA walks: units 0 .. full-1 are whole tiles, the rest (tile, split) pairs of the remaining tiles.
struct Sched {
    int tiles_m, tiles_n, tiles, full, splits, units, kblocks, kper;
    float inv_band;         // 1 / (tiles of a band)
    float* part;            // [units - full][rows of a tile][BN]
};

struct Unit {
    int m0, n0, kb0, kb1, slot;      // slot < 0: a whole tile
};

// Tiles are taken in bands of eight rows of tiles, down each band's columns: what runs at one time then spans about as
// many rows as columns, and reads the least of either operand.
constexpr int kBand = 8;
__device__ __forceinline__ void place_of_tile(const Sched& s, int tile, int* m, int* n) {
    const int size = kBand * s.tiles_n;
    // tile / size: an estimate that is put right, shorter than the division that every warp would wait for at every tile
    int band = (int)((float)tile * s.inv_band), in = tile - band * size;
    while (in < 0) { --band; in += size; }
    while (in >= size) { ++band; in -= size; }
    const int first = band * kBand, high = s.tiles_m - first;
    if (high >= kBand) {
        *m = first + in % kBand;
        *n = in / kBand;
    } else {
        *m = first + in % high;
        *n = in / high;
    }
}

template <int BN>
__device__ __forceinline__ Unit unit_of(const Sched& s, int u) {
    Unit r;
    int tile = u;
    r.kb0 = 0;
    r.kb1 = s.kblocks;
    r.slot = -1;
    if (u >= s.full) {
        r.slot = u - s.full;
        tile = s.full + r.slot / s.splits;
        r.kb0 = (r.slot % s.splits) * s.kper;
        r.kb1 = min(r.kb0 + s.kper, s.kblocks);
    }
    place_of_tile(s, tile, &r.m0, &r.n0);
    r.m0 *= Cfg<BN>::kRows;
    r.n0 *= BN;
    return r;
}

// W words of a row in registers to and from memory, E elements of 2 or 4 bytes of which the first `left` count.  vec: 2 where
// the address is a multiple of 32 bytes (one instruction a sector), 1 of 16, 0 of an element.
template <int W, typename E>
__device__ __forceinline__ void store_row(const uint32_t* w, E* p, int left, int vec) {
    constexpr int per = 4 / sizeof(E);
    if (left >= W * per && vec) {
        if (vec == 2) {
#pragma unroll
            for (int i = 0; i < W; i += 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + i * per), "r"(w[i]), "r"(w[i + 1]),
                             "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                             : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < W; i += 4)
                *reinterpret_cast<uint4*>(p + i * per) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (per == 1) {
            if (i < left) reinterpret_cast<uint32_t*>(p)[i] = w[i];
        } else {
            if (2 * i < left) p[2 * i] = (E)w[i];
            if (2 * i + 1 < left) p[2 * i + 1] = (E)(w[i] >> 16);
        }
    }
}
template <int W, typename E>
__device__ __forceinline__ void load_row(uint32_t* w, const E* p, int left, int vec) {
    constexpr int per = 4 / sizeof(E);
    if (left >= W * per && vec) {
        if (vec == 2) {
#pragma unroll
            for (int i = 0; i < W; i += 8)
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]),
                               "=r"(w[i + 6]), "=r"(w[i + 7])
                             : "l"(p + i * per)
                             : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const uint4 q = *reinterpret_cast<const uint4*>(p + i * per);
                w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (per == 1) {
            w[i] = i < left ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
        } else {
            w[i] = 2 * i < left ? (uint32_t)p[2 * i] : 0u;
            if (2 * i + 1 < left) w[i] |= (uint32_t)p[2 * i + 1] << 16;
        }
    }
}

// FINE: GELU for an fp32 result, and no other activation; its code beside the others slows all of them (without an activation
// 38,400 x 1024 x 4096 takes 270 us in long runs, and 285 with it).
template <typename T, int BN, bool AMN, bool BMN, bool FINE>
__global__ void __launch_bounds__(kGemmThreads, 1)
    k_gemm(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const int M, const int N,
           const __grid_constant__ Sched sched, const __grid_constant__ Out o, int32_t* status) {
    using C = Cfg<BN>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBars);
    uint64_t* empty = full + C::kStages;
    uint64_t* acc_full = empty + C::kStages;       // 2
    uint64_t* acc_empty = acc_full + 2;            // 2
    uint64_t* drain = acc_empty + 2;
    uint32_t* slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, (C::kPair ? 2 : 1) * kEpiWarps);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (C::kPair) tmem_alloc_pair(slot, 2 * BN);
        else tmem_alloc(slot, 2 * BN);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (C::kPair) cluster_sync();             // the other CTA's barriers are ready too
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *slot, 0);
    const int rank = C::kPair ? (int)cluster_rank() : 0;
    const int first = C::kPair ? blockIdx.x >> 1 : blockIdx.x, step = C::kPair ? gridDim.x >> 1 : gridDim.x;
    pdl_begin();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int u = first; u < sched.units && ok; u += step) {
                const Unit t = unit_of<BN>(sched, u);
                const int m0 = t.m0 + rank * kBM, n0 = t.n0 + rank * C::kOwnN;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                    const int st = it % C::kStages;
                    if (!mbar_wait(empty + st, ((it / C::kStages) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx(full + st, (C::kPair ? 2 : 1) * C::kStage);
                    const uint32_t a = smem_u32(smem + st * C::kStage), b = a + C::kA;
                    const uint32_t bar = C::kPair ? even_bar(full + st) : 0;
                    auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y) {
                        if constexpr (C::kPair) tma_tile2d_pair(to, map, x, y, bar);
                        else tma_tile2d(to, map, x, y, full + st);
                    };
                    if constexpr (AMN) {
#pragma unroll
                        for (int i = 0; i < kBM / 64; ++i) load(a + i * 8192, &ma, m0 + 64 * i, kb * kBK);
                    } else {
                        load(a, &ma, kb * kBK, m0);
                    }
                    if constexpr (BMN) {
#pragma unroll
                        for (int i = 0; i < C::kOwnN / 64; ++i) load(b + i * 8192, &mb, n0 + 64 * i, kb * kBK);
                    } else {
                        load(b, &mb, kb * kBK, n0);
                    }
                }
            }
            if (!ok) {
                *abort_flag = 1;
                flag(status, PMG_ERR_TIMEOUT);
            }
        }
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t idesc = idesc16(Elem<T>::kFmt, C::kRows, BN, AMN, BMN);
        const uint32_t lead = elect_one();
        uint32_t it = 0, k = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, ph, abort_flag)); };
        for (int u = first; u < sched.units && ok; u += step, ++k) {
            const Unit t = unit_of<BN>(sched, u);
            const uint32_t buf = k & 1u, d = tmem + buf * BN;
            ok = wait(acc_empty + buf, ((k >> 1) & 1u) ^ 1u);
            if (!ok) break;
            tc_fence_after();
            for (int kb = t.kb0; kb < t.kb1; ++kb, ++it) {
                const int st = it % C::kStages;
                ok = wait(full + st, (it / C::kStages) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem_u32(smem + st * C::kStage);
                const uint32_t a = desc_lo(at, AMN ? 8192 : 16), b = desc_lo(at + C::kA, BMN ? 8192 : 16);
#pragma unroll
                for (int kk = 0; kk < kBK / 16; ++kk) {
                    const uint32_t da = a + kk * (AMN ? 128 : 2), db = b + kk * (BMN ? 128 : 2), acc = (kb > t.kb0 || kk > 0) ? 1u : 0u;
                    if constexpr (C::kPair) mma16_pair(lead, d, da, db, idesc, acc);
                    else mma16(lead, d, da, db, idesc, acc);
                }
                if constexpr (C::kPair) commit_pair_if(lead, empty + st);
                else mma_commit_if(lead, empty + st);
            }
            if (!ok) break;
            if constexpr (C::kPair) commit_pair_if(lead, acc_full + buf);
            else mma_commit_if(lead, acc_full + buf);
        }
        if (lane == 0) {
            if (!ok) flag(status, PMG_ERR_TIMEOUT);
            if (!ok || *abort_flag) {
                *abort_flag = 1;
                drain_mma<C::kPair>(drain);
            }
        }
        __syncwarp();
    } else if (warp >= kFirstEpi) {
        // Warp w of the sixteen takes the quarter of the rows that it can read (w mod 4) and a quarter of the columns, a
        // lane a row.  Rows go from registers to memory in sectors of 32 bytes, not by way of shared memory, whose
        // bandwidth the products and their loads fill (64 + 64 of 128 bytes a cycle).
        constexpr int kOwn = BN / 4, kChunk = kOwn < 32 ? kOwn : 32;
        const int ew = warp - kFirstEpi, quarter = warp & 3, group = ew >> 2;
        T* bias_s = reinterpret_cast<T*>(smem + C::kStages * C::kStage) + ew * kOwn;
        uint32_t k = 0;
        bool ok = true;
        // A tile's bias comes while the tile before is worked on.
        constexpr int kBiasRegs = (kOwn + 31) / 32;
        T bias_r[kBiasRegs];
        auto ask_bias = [&](const Unit& t) {
            if (!o.bias || t.slot >= 0) return;
#pragma unroll
            for (int i = 0; i < kBiasRegs; ++i) {
                const int c = 32 * i + lane, n = t.n0 + group * kOwn + c;
                bias_r[i] = c < kOwn && n < N ? static_cast<const T*>(o.bias)[n] : Elem<T>::from(0.0f);
            }
        };
        Unit t = unit_of<BN>(sched, min(first, sched.units - 1)), next;
        ask_bias(t);
        for (int u = first; u < sched.units; u += step, ++k, t = next) {
            next = unit_of<BN>(sched, min(u + step, sched.units - 1));
            const uint32_t buf = k & 1u;
            const int in = quarter * 32 + lane, m = t.m0 + rank * kBM + in;
            const bool whole = t.slot < 0, row = m < M;
            const int own = min(kOwn, N - t.n0 - group * kOwn);            // columns of this warp within the matrix
            if (whole && o.bias) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kBiasRegs; ++i)
                    if (32 * i + lane < kOwn) bias_s[32 * i + lane] = bias_r[i];
                __syncwarp();
            }
            ask_bias(next);
            bool waited = false;
#pragma unroll 1
            for (int c0 = 0; c0 < own || !waited; c0 += kChunk) {
                const int c = group * kOwn + c0, n = t.n0 + c, left = N - n;
                const bool add = whole && o.resid && row;
                uint32_t res[kChunk];                         // ahead of the accumulators
                if (add) {
                    if (o.f32) load_row<kChunk>(res, static_cast<const float*>(o.resid) + (int64_t)m * o.ldr + n, left, o.vec);
                    else load_row<kChunk / 2>(res, static_cast<const uint16_t*>(o.resid) + (int64_t)m * o.ldr + n, left, o.vec);
                }
                if (!waited) {
                    waited = true;
                    ok = __all_sync(0xffffffffu, mbar_wait(acc_full + buf, (k >> 1) & 1u, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                }
                const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + buf * BN + c;
                float v[kChunk];
                if constexpr (kChunk == 32) tmem_ld32(src, reinterpret_cast<uint32_t*>(v));
                else tmem_ld16(src, *reinterpret_cast<uint32_t (*)[16]>(v));
                tmem_wait_ld();
                if (c0 + kChunk >= own) {                     // all that this warp wants is in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (C::kPair) arrive_even(acc_empty + buf);
                        else mbar_arrive(acc_empty + buf);
                    }
                }
                if (!whole) {
                    float* p = sched.part + ((int64_t)t.slot * C::kRows + rank * kBM + in) * BN + c;
                    store_row<kChunk>(reinterpret_cast<uint32_t*>(v), p, row ? left : 0,
                                      reinterpret_cast<uintptr_t>(sched.part) & 31 ? 1 : 2);
                    continue;
                }
                if (o.bias) {
#pragma unroll
                    for (int i = 0; i < kChunk; i += 8) {
                        const uint4 q = *reinterpret_cast<const uint4*>(bias_s + c0 + i);
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = Elem<T>::unpack(w[e]);
                            v[i + 2 * e] += f.x;
                            v[i + 2 * e + 1] += f.y;
                        }
                    }
                }
                uint32_t h[kChunk / 2];
                if (o.pre) {
#pragma unroll
                    for (int i = 0; i < kChunk; i += 2) h[i / 2] = Elem<T>::pack(v[i], v[i + 1]);
                    store_row<kChunk / 2>(h, static_cast<uint16_t*>(o.pre) + (int64_t)m * o.ldp + n, row ? left : 0, o.vec);
                }
                if constexpr (FINE) {
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) v[i] = gelu_fine(v[i]);
                } else {
                    activate<T, kChunk>(o.act, false, v);
                }
                if (o.f32) {
                    if (add) {
#pragma unroll
                        for (int i = 0; i < kChunk; ++i) v[i] += __uint_as_float(res[i]);
                    }
                    store_row<kChunk>(reinterpret_cast<uint32_t*>(v), static_cast<float*>(o.y) + (int64_t)m * o.ldy + n,
                                      row ? left : 0, o.vec);
                } else {
                    if (add) {
#pragma unroll
                        for (int i = 0; i < kChunk; i += 2) {
                            const float2 f = Elem<T>::unpack(res[i / 2]);
                            v[i] += f.x;
                            v[i + 1] += f.y;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kChunk; i += 2) h[i / 2] = Elem<T>::pack(v[i], v[i + 1]);
                    store_row<kChunk / 2>(h, static_cast<uint16_t*>(o.y) + (int64_t)m * o.ldy + n, row ? left : 0, o.vec);
                }
            }
            if (!ok) break;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            flag(status, PMG_ERR_TIMEOUT);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (C::kPair) cluster_sync();             // neither leaves while the other may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        if constexpr (C::kPair) tmem_dealloc_pair(tmem, 2 * BN);
        else tmem_dealloc(tmem, 2 * BN);
    }
}

template <typename T, int BN>
__global__ void __launch_bounds__(256) k_split_sum(const __grid_constant__ Sched s, const int M, const int N,
                                                   const __grid_constant__ Out o) {
    pdl_begin();
    constexpr int kRows = Cfg<BN>::kRows, per_tile = kRows * BN / 8;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int rest = i / per_tile, tile = s.full + rest, e = (i % per_tile) * 8;
    if (tile >= s.tiles) return;
    const int r = e / BN, c = e % BN;
    int tm, tn;
    place_of_tile(s, tile, &tm, &tn);
    const int m = tm * kRows + r, n = tn * BN + c;
    if (m >= M || n >= N) return;
    float z[8] = {};
    const float* p = s.part + ((int64_t)rest * s.splits * kRows + r) * BN + c;
    for (int k = 0; k < s.splits; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        z[0] += a.x; z[1] += a.y; z[2] += a.z; z[3] += a.w;
        z[4] += b.x; z[5] += b.y; z[6] += b.z; z[7] += b.w;
        p += kRows * BN;
    }
    finish8<T>(o, m, n, N, z);
}

// ----------------------------------------------------------------------------------------------------------------- //
// Backwards: dz and the bias gradient; row packing
// ----------------------------------------------------------------------------------------------------------------- //
constexpr int kStripCols = 256, kStripRows = 8;       // a block's columns; rows at a time

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = Elem<T>::unpack(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

// dz = dy act'(z) rounded to T into dst (null: not wanted) with its row padding zeroed, and this block's column sums of
// the unrounded dz into part [row blocks][N] (null: not wanted).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 4) k_act_grad(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ pre,
                                                  int64_t ldp, int64_t M, int N, int act, T* __restrict__ dst,
                                                  int64_t ldd, int padded, int64_t rows_per_block,
                                                  float* __restrict__ part) {
    pdl_begin();
    __shared__ float sm[kStripRows][kStripCols];
    const int cg = threadIdx.x & 31, rg = threadIdx.x >> 5, n = blockIdx.x * kStripCols + cg * 8;
    const int64_t r0 = blockIdx.y * rows_per_block, r1 = min(r0 + rows_per_block, M);
    float acc[8] = {};
    const bool vec = VEC && n + 8 <= N;
    auto row = [&](const T* p, int64_t ld, int64_t m) {               // 8 values, zero beyond the matrix
        if (m >= r1) return make_uint4(0, 0, 0, 0);
        if (vec) return *reinterpret_cast<const uint4*>(p + m * ld + n);
        uint32_t w[4] = {0, 0, 0, 0};
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p + m * ld + n);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < N) w[i >> 1] |= (uint32_t)q[i] << (16 * (i & 1));
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    if (n < padded) {
        constexpr int U = 2;        // rows on their way at once; 4 of them leave half the warps, and took 4 us longer
        for (int64_t m0 = r0 + rg; m0 < r1; m0 += U * kStripRows) {
            uint4 dr[U], zr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) dr[u] = row(dy, ldy, m0 + u * kStripRows);
            if (pre) {
#pragma unroll
                for (int u = 0; u < U; ++u) zr[u] = row(pre, ldp, m0 + u * kStripRows);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t m = m0 + u * kStripRows;
                float g[8], z[8];
                unpack8<T>(dr[u], g);
                if (pre) {
                    unpack8<T>(zr[u], z);
                    times_slope(act, g, z);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += g[i];
                if (dst && m < r1) {
                    *reinterpret_cast<uint4*>(dst + m * ldd + n) =
                        make_uint4(Elem<T>::pack(g[0], g[1]), Elem<T>::pack(g[2], g[3]), Elem<T>::pack(g[4], g[5]), Elem<T>::pack(g[6], g[7]));
                }
            }
        }
    }
    if (part == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sm[rg][cg * 8 + i] = acc[i];
    __syncthreads();
    const int col = blockIdx.x * kStripCols + threadIdx.x;
    if (col < N) {
        float v = 0.0f;
#pragma unroll
        for (int r = 0; r < kStripRows; ++r) v += sm[r][threadIdx.x];
        part[(int64_t)blockIdx.y * N + col] = v;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_col_sum(const float* __restrict__ part, int blocks, int N, T* __restrict__ out) {
    pdl_begin();
    __shared__ float sm[8][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    float v = 0.0f;
    if (col < N)
        for (int b = strand; b < blocks; b += 8) v += part[(int64_t)b * N + col];
    sm[strand][threadIdx.x & 31] = v;
    __syncthreads();
    if (strand == 0 && col < N) {
        float t = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) t += sm[s][threadIdx.x];
        out[col] = Elem<T>::from(t);
    }
}

// Rows copied to 16-byte-aligned rows of `ldd` values, padding zeroed: one or two matrices of the same width.
struct Pack {
    const uint16_t* src[2];
    uint16_t* dst[2];
    int64_t lds[2], rows[2], ldd;
    int cols;
};
__global__ void __launch_bounds__(256) k_pack_rows(const __grid_constant__ Pack a) {
    pdl_begin();
    const int groups = (int)(a.ldd / 8);
    const int64_t n0 = a.rows[0] * groups, n = n0 + a.rows[1] * groups;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int m = i >= n0;
        const int64_t j = m ? i - n0 : i, r = j / groups;
        const int c = (int)(j - r * groups) * 8;
        const uint16_t* p = a.src[m] + r * a.lds[m] + c;
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < a.cols) w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
        *reinterpret_cast<uint4*>(a.dst[m] + r * a.ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ----------------------------------------------------------------------------------------------------------------- //
// Host side
// ----------------------------------------------------------------------------------------------------------------- //
int64_t round8(int64_t v) { return (v + 7) & ~(int64_t)7; }
size_t round256(size_t v) { return (v + 255) & ~(size_t)255; }
bool tma_ok(const void* p, int64_t ld) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(ld & 7); }

constexpr int kFewRows = 32;

// How a product is cut.  In cycles of one SM, measured: a K block takes 512 with tiles of 256 x 256 by two CTAs (the
// products' own time) and 390 with narrower ones (the loads'); the epilogue of the last tile about 25 a column; a last wave
// cut along K costs its second kernel, about 7000.  The gradient of a 4096 x 1024 weight over 9600 rows takes 57 us with
// tiles of 256 (64 on 74 pairs), 76 with 128; 1200 x 1024 x 1024 takes 8.3 us with 80 tiles of 128, 12 with 20 of 256;
// 600 x 1024 x 1024 takes 7.3 us with tiles of 64 columns, 8.0 with 128.
Sched schedule(int64_t M, int64_t N, int64_t K, int bn, int64_t* cost) {
    Sched s{};
    s.tiles_n = (int)((N + bn - 1) / bn);
    const int rows = bn == 256 ? 2 * kBM : kBM, slots = bn == 256 ? kNumSMs / 2 : kNumSMs;      // two CTAs a tile, or one
    s.tiles_m = (int)((M + rows - 1) / rows);
    s.tiles = s.tiles_m * s.tiles_n;
    s.inv_band = 1.0f / (float)(kBand * s.tiles_n);
    s.kblocks = (int)((K + kBK - 1) / kBK);
    s.full = s.tiles;
    s.splits = 1;
    s.kper = s.kblocks;
    const int64_t block = bn == 256 ? 512 : 390, epilogue = 25 * bn;
    const int waves = s.tiles / slots, rest = s.tiles % slots;
    *cost = (waves + (rest > 0)) * s.kblocks * block + epilogue;
    // at least two splits of four blocks each
    const int splits = rest ? std::min({slots / rest, s.kblocks / 4, 16}) : 1;
    if (splits >= 2) {
        const int kper = (s.kblocks + splits - 1) / splits;
        const int64_t cut = (waves * s.kblocks + kper) * block + epilogue + 7000;
        if (cut < *cost) {
            *cost = cut;
            s.full = s.tiles - rest;
            s.kper = kper;
            s.splits = (s.kblocks + kper - 1) / kper;
        }
    }
    s.units = s.full + (s.tiles - s.full) * s.splits;
    return s;
}

// Tile width and schedule of least cost.
int choose(int64_t M, int64_t N, int64_t K, Sched* s) {
    int best = 0;
    int64_t least = 0;
    for (int bn : {256, 128, 64}) {
        int64_t cost;
        const Sched t = schedule(M, N, K, bn, &cost);
        if (best == 0 || cost < least) {
            best = bn;
            least = cost;
            *s = t;
        }
    }
    return best;
}

size_t part_bytes(int64_t M, int64_t N, int64_t K) {
    Sched s;
    const int bn = choose(M, N, K, &s);
    return (size_t)(s.units - s.full) * (bn == 256 ? 2 * kBM : kBM) * bn * sizeof(float);
}

template <typename T, int BN, bool AMN, bool BMN, bool FINE>
int gemm_bn(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K, const Out& o,
            Sched s, int32_t* status, cudaStream_t st) {
    using C = Cfg<BN>;
    static bool attr_set[64] = {};
    int dev = 0;
    PMG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return PMG_ERR_UNSUPPORTED;
    if (!attr_set[dev]) {
        PMG_CUDA_TRY(cudaFuncSetAttribute(k_gemm<T, BN, AMN, BMN, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        attr_set[dev] = true;
    }
    CUtensorMap ma, mb;
    const uint64_t da[2] = {(uint64_t)(AMN ? M : K), (uint64_t)(AMN ? K : M)}, sa[1] = {(uint64_t)lda * 2};
    const uint64_t db[2] = {(uint64_t)(BMN ? N : K), (uint64_t)(BMN ? K : N)}, sb[1] = {(uint64_t)ldb * 2};
    const uint32_t ba[2] = {64, (uint32_t)(AMN ? kBK : kBM)}, bb[2] = {64, (uint32_t)(BMN ? kBK : C::kOwnN)};
    int rc = make_tensor_map16(&ma, A, 2, da, sa, ba);
    if (rc != PMG_OK) return rc;
    rc = make_tensor_map16(&mb, B, 2, db, sb, bb);
    if (rc != PMG_OK) return rc;
    constexpr int kCtas = C::kPair ? 2 : 1;
    rc = launch_after<kCtas>(k_gemm<T, BN, AMN, BMN, FINE>, dim3(std::min(s.units, kNumSMs / kCtas) * kCtas), kGemmThreads, C::kSmem, st,
                             ma, mb, (int)M, (int)N, s, o, status);
    if (rc != PMG_OK) return rc;
    if (s.full < s.tiles) {
        const int64_t threads = (int64_t)(s.tiles - s.full) * (C::kRows * BN / 8);
        return launch_after(k_split_sum<T, BN>, dim3((unsigned)((threads + 255) / 256)), 256, 0, st, s, (int)M, (int)N, o);
    }
    return PMG_OK;
}

template <typename T, bool AMN, bool BMN, bool FINE = false>
int gemm(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N, int64_t K, const Out& o,
         float* part, int32_t* status, cudaStream_t st) {
    Sched c;
    const int bn = choose(M, N, K, &c);
    c.part = part;
    switch (bn) {
        case 256: return gemm_bn<T, 256, AMN, BMN, FINE>(A, lda, B, ldb, M, N, K, o, c, status, st);
        case 128: return gemm_bn<T, 128, AMN, BMN, FINE>(A, lda, B, ldb, M, N, K, o, c, status, st);
        default: return gemm_bn<T, 64, AMN, BMN, FINE>(A, lda, B, ldb, M, N, K, o, c, status, st);
    }
}

// Copies of those of two matrices of `cols` columns that TMA cannot read, at `ws`, which moves on; they are replaced.
struct Matrix {
    const void* p;
    int64_t ld, rows;
};
int pack(Matrix* x, Matrix* w, int64_t cols, uint8_t*& ws, cudaStream_t s) {
    Pack a{};
    a.ldd = round8(cols);
    a.cols = (int)cols;
    int n = 0;
    int64_t groups = 0;
    for (Matrix* m : {x, w}) {
        if (!m || tma_ok(m->p, m->ld)) continue;
        a.src[n] = static_cast<const uint16_t*>(m->p);
        a.dst[n] = reinterpret_cast<uint16_t*>(ws);
        a.lds[n] = m->ld;
        a.rows[n] = m->rows;
        groups += m->rows * (a.ldd / 8);
        m->p = ws;
        m->ld = a.ldd;
        ws += round256((size_t)m->rows * a.ldd * 2);
        ++n;
    }
    if (n == 0) return PMG_OK;
    return launch_after(k_pack_rows, dim3((unsigned)std::min<int64_t>((groups + 255) / 256, kNumSMs * 16)), 256, 0, s, a);
}

template <typename T, int NT>
int rows_nt(const void* x, int64_t ldx, const void* w, int64_t ldw, int M, int N, int K, const Out& o, cudaStream_t s) {
    const bool aligned = tma_ok(x, ldx) && tma_ok(w, ldw) && K % 8 == 0;
    int warps = std::min(16, std::max(4, (K + 127) / 128));
    while (warps & (warps - 1)) warps &= warps - 1;
    const size_t smem = (size_t)warps * kRowsCols * 8 * NT * sizeof(float);
    const int grid = (N + kRowsCols - 1) / kRowsCols;
    const uint16_t *xp = static_cast<const uint16_t*>(x), *wp = static_cast<const uint16_t*>(w);
    if (aligned) k_rows<T, NT, true><<<grid, 32 * warps, smem, s>>>(xp, ldx, wp, ldw, M, N, K, o);
    else k_rows<T, NT, false><<<grid, 32 * warps, smem, s>>>(xp, ldx, wp, ldw, M, N, K, o);
    PMG_LAUNCH_CHECK();
    return PMG_OK;
}

// What store_row may use: 2, 1 or 0 by the least aligned of the row starts.
int vec_ok(const Out& o) {
    uintptr_t bits = 0;
    auto see = [&](const void* p, int64_t ld, int esz) {
        if (p) bits |= reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * esz);
    };
    see(o.y, o.ldy, o.f32 ? 4 : 2);
    see(o.resid, o.ldr, o.f32 ? 4 : 2);
    see(o.pre, o.ldp, 2);
    return bits & 15 ? 0 : bits & 31 ? 1 : 2;
}

template <typename T>
int linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, Out o, uint8_t* ws,
           int32_t* status, cudaStream_t s) {
    o.vec = vec_ok(o);
    if (M <= 8) return rows_nt<T, 1>(x, ldx, w, ldw, (int)M, (int)N, (int)K, o, s);
    if (M <= 16) return rows_nt<T, 2>(x, ldx, w, ldw, (int)M, (int)N, (int)K, o, s);
    if (M <= kFewRows) return rows_nt<T, 4>(x, ldx, w, ldw, (int)M, (int)N, (int)K, o, s);
    Matrix mx{x, ldx, M}, mw{w, ldw, N};
    const int rc = pack(&mx, &mw, K, ws, s);
    if (rc != PMG_OK) return rc;
    const auto product = o.act == PMG_ACT_GELU && o.f32 ? gemm<T, false, false, true> : gemm<T, false, false>;
    return product(mx.p, mx.ld, mw.p, mw.ld, M, N, K, o, reinterpret_cast<float*>(ws), status, s);
}

struct GradPlan {
    int64_t row_blocks, rows_per_block;
    bool dz;                 // a rounded (or packed) dz is stored
};

GradPlan grad_plan(int64_t M, int64_t N, bool act, bool dy_ok) {
    GradPlan p;
    const int64_t strips = (N + kStripCols - 1) / kStripCols;
    const int64_t want = std::max<int64_t>(1, kNumSMs * 4 / strips);      // blocks for one wave, four a SM
    p.rows_per_block = std::max<int64_t>(kStripRows * 2, (M + want - 1) / want);
    p.row_blocks = std::max<int64_t>(1, (M + p.rows_per_block - 1) / p.rows_per_block);
    p.dz = act || !dy_ok;
    return p;
}

template <typename T>
int linear_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
                int64_t N, int64_t K, const void* pre, int64_t ldp, int act, void* dx, int64_t lddx, void* dw,
                int64_t lddw, void* db, uint8_t* ws, int32_t* status, cudaStream_t s) {
    const bool has_act = act != PMG_ACT_NONE, products = dx || dw;
    const GradPlan p = grad_plan(M, N, has_act, tma_ok(dy, lddy));
    const void* dz = dy;
    int64_t lddz = lddy;
    if (db || (p.dz && products)) {
        T* dst = nullptr;
        if (p.dz && products) {
            dst = reinterpret_cast<T*>(ws);
            lddz = round8(N);
            dz = dst;
            ws += round256((size_t)M * lddz * 2);
        }
        float* part = nullptr;
        if (db) {
            part = reinterpret_cast<float*>(ws);
            ws += round256((size_t)p.row_blocks * N * sizeof(float));
        }
        const dim3 grid((unsigned)((N + kStripCols - 1) / kStripCols), (unsigned)p.row_blocks);
        const bool vec = tma_ok(dy, lddy) && (!has_act || tma_ok(pre, ldp));
        const T *dyp = static_cast<const T*>(dy), *prep = has_act ? static_cast<const T*>(pre) : nullptr;
        if (vec) k_act_grad<T, true><<<grid, 256, 0, s>>>(dyp, lddy, prep, ldp, M, (int)N, act, dst, lddz, (int)round8(N), p.rows_per_block, part);
        else k_act_grad<T, false><<<grid, 256, 0, s>>>(dyp, lddy, prep, ldp, M, (int)N, act, dst, lddz, (int)round8(N), p.rows_per_block, part);
        PMG_LAUNCH_CHECK();
        if (db) {
            const int rc = launch_after(k_col_sum<T>, dim3((unsigned)((N + 31) / 32)), 256, 0, s, (const float*)part,
                                        (int)p.row_blocks, (int)N, static_cast<T*>(db));
            if (rc != PMG_OK) return rc;
        }
    }
    Matrix mx{x, ldx, M}, mw{w, ldw, N};
    const int rc = pack(dw ? &mx : nullptr, dx ? &mw : nullptr, K, ws, s);
    if (rc != PMG_OK) return rc;
    Out o{};
    if (dx) {
        o.y = dx;
        o.ldy = lddx;
        o.vec = vec_ok(o);
        const int rc2 = gemm<T, false, true>(dz, lddz, mw.p, mw.ld, M, K, N, o, reinterpret_cast<float*>(ws), status, s);
        if (rc2 != PMG_OK) return rc2;
    }
    if (dw) {
        o.y = dw;
        o.ldy = lddw;
        o.vec = vec_ok(o);
        const int rc2 = gemm<T, true, true>(dz, lddz, mx.p, mx.ld, N, K, M, o, reinterpret_cast<float*>(ws), status, s);
        if (rc2 != PMG_OK) return rc2;
    }
    return PMG_OK;
}

int check_linear(int dtype, int64_t M, int64_t N, int64_t K, int act) {
    if (dtype != PMG_F16 && dtype != PMG_BF16) return PMG_ERR_UNSUPPORTED;
    if (M < 0 || N < 1 || K < 1 || act < PMG_ACT_NONE || act > PMG_ACT_GELU) return PMG_ERR_BAD_ARG;
    if (M > (int64_t)1 << 30 || N > 1 << 20 || K > 1 << 20) return PMG_ERR_UNSUPPORTED;
    if (((M + kBM - 1) / kBM) * ((std::max(N, K) + 63) / 64) > (int64_t)1 << 30) return PMG_ERR_UNSUPPORTED;
    return PMG_OK;
}

}  // namespace
}  // namespace pmg

using namespace pmg;

extern "C" size_t pmg_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t pack_x, int32_t pack_w) {
    if (M <= kFewRows || N < 1 || K < 1) return 0;
    return (pack_x ? round256((size_t)M * round8(K) * 2) : 0) + (pack_w ? round256((size_t)N * round8(K) * 2) : 0) +
           part_bytes(M, N, K);
}

extern "C" int pmg_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int32_t dtype, int64_t M, int64_t N,
                          int64_t K, const void* bias, int32_t act, const void* residual, int64_t ldr, int32_t out_f32,
                          void* y, int64_t ldy, void* pre, int64_t ldp, void* workspace, size_t workspace_bytes,
                          int32_t* status, void* stream) {
    const int rc = check_linear(dtype, M, N, K, act);
    if (rc != PMG_OK) return rc;
    if (M == 0) return PMG_OK;
    if (!x || !w || !y || ldx < K || ldw < K || ldy < N || (residual && ldr < N) || (pre && ldp < N)) return PMG_ERR_BAD_ARG;
    const size_t need = pmg_linear_workspace_bytes(M, N, K, !tma_ok(x, ldx), !tma_ok(w, ldw));
    if (workspace_bytes < need || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))) return PMG_ERR_BAD_ARG;
    Out o{};
    o.bias = bias; o.resid = residual; o.y = y; o.pre = pre;
    o.ldr = ldr; o.ldy = ldy; o.ldp = ldp; o.act = act; o.f32 = out_f32 != 0;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    return dtype == PMG_BF16 ? linear<__nv_bfloat16>(x, ldx, w, ldw, M, N, K, o, ws, status, as_stream(stream))
                             : linear<__half>(x, ldx, w, ldw, M, N, K, o, ws, status, as_stream(stream));
}

extern "C" size_t pmg_linear_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t act, int32_t pack_dy,
                                                  int32_t pack_x, int32_t pack_w, int32_t bias_grad) {
    if (M < 1 || N < 1 || K < 1) return 0;
    const GradPlan p = grad_plan(M, N, act != PMG_ACT_NONE, !pack_dy);
    const size_t dz = p.dz ? round256((size_t)M * round8(N) * 2) : 0;
    const size_t db = bias_grad ? round256((size_t)p.row_blocks * N * sizeof(float)) : 0;
    const size_t packed = (pack_w ? round256((size_t)N * round8(K) * 2) : 0) + (pack_x ? round256((size_t)M * round8(K) * 2) : 0);
    return dz + db + packed + std::max(part_bytes(M, K, N), part_bytes(N, K, M));
}

extern "C" int pmg_linear_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                               int32_t dtype, int64_t M, int64_t N, int64_t K, const void* pre, int64_t ldp,
                               int32_t act, void* dx, int64_t lddx, void* dw, int64_t lddw, void* db, void* workspace,
                               size_t workspace_bytes, int32_t* status, void* stream) {
    const int rc = check_linear(dtype, M, N, K, act);
    if (rc != PMG_OK) return rc;
    cudaStream_t s = as_stream(stream);
    if (M == 0) {                                     // no rows: the sums over rows are zero
        if (dw) PMG_CUDA_TRY(cudaMemset2DAsync(dw, (size_t)lddw * 2, 0, (size_t)K * 2, (size_t)N, s));
        if (db) PMG_CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)N * 2, s));
        return PMG_OK;
    }
    if (!dy || lddy < N || (act != PMG_ACT_NONE && (!pre || ldp < N)) || (dx && (!w || ldw < K || lddx < K)) ||
        (dw && (!x || ldx < K || lddw < K)))
        return PMG_ERR_BAD_ARG;
    const size_t need = pmg_linear_grad_workspace_bytes(M, N, K, act, !tma_ok(dy, lddy), dw && !tma_ok(x, ldx),
                                                        dx && !tma_ok(w, ldw), db != nullptr);
    if (workspace_bytes < need || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))) return PMG_ERR_BAD_ARG;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    return dtype == PMG_BF16
               ? linear_grad<__nv_bfloat16>(dy, lddy, x, ldx, w, ldw, M, N, K, pre, ldp, act, dx, lddx, dw, lddw, db, ws, status, s)
               : linear_grad<__half>(dy, lddy, x, ldx, w, ldw, M, N, K, pre, ldp, act, dx, lddx, dw, lddw, db, ws, status, s);
}
