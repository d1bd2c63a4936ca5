// ffn_kernels.hip -- the gated feed-forward block of a trainable backbone (pose_estimation/train.py:97-119 back-propagates through
// pose_estimation/backbone.py:12-14), forward and backward:
//     [g | u] = x W12^T + b12,   h = act(g) u,   y = h W3^T + b3                    x [M][D], W12 [2H][D], W3 [O][H]
//     q = act(g), p = u act'(g):  dh = dy W3,  dg = dh p,  du = dh q
//     dx = [dg | du] W12,  dW12 = [dg | du]^T x,  dW3 = dy^T h,  db12 = sum_m [dg | du],  db3 = sum_m dy
// Six matrix products; both projections, the activation and the product of the first are ONE launch (the gate and up columns of a
// hidden unit sit in the same lane's accumulators), and so are dh and the two factors' products.
// The forward pass keeps h in the activations' type (it is the second product's operand) and p, q in fp32: rounding them too would
// add a third rounding between dy and dx (measured against 64 bits: 2.1 roundings' worth instead of 1.4).
#include "block_launch.h"
#include "block_types.h"

#include <algorithm>

namespace {

enum { ACT_SILU = 0, ACT_GELU = 1 };

// act(g) and act'(g)
template <bool EXACT>
__device__ __forceinline__ void activation(int act, float g, float& f, float& df) {
    if (act == ACT_SILU) {                         // s = 1 / (1 + e^-g), act = g s, act' = s (1 + g (1 - s))
        const float s = 1.0f / (1.0f + (EXACT ? expf(-g) : __expf(-g)));
        f = g * s;
        df = s * fmaf(g, 1.0f - s, 1.0f);
    } else {                                       // c = (1 + erf(g / sqrt 2)) / 2, act = g c, act' = c + g e^(-g^2/2) / sqrt(2 pi)
        const float c = 0.5f * erfcf(-0.70710678118654752440f * g);
        f = g * c;
        df = fmaf(g * 0.39894228040143267794f, EXACT ? expf(-0.5f * g * g) : __expf(-0.5f * g * g), c);
    }
}

// matrix-core element of a type and its product; fp32 runs as three bf16 pieces a = a0 + a1 + a2 (8 bits each, by truncation: exact) and
// the six products whose weight is above 2^-24
template <class T> struct Mat { typedef __bf16 e; static constexpr int P = 3; };
template <> struct Mat<__bf16> { typedef __bf16 e; static constexpr int P = 1; };
template <> struct Mat<_Float16> { typedef _Float16 e; static constexpr int P = 1; };
typedef __bf16 vb8 __attribute__((ext_vector_type(8)));
typedef _Float16 vh8 __attribute__((ext_vector_type(8)));
template <class E> struct V8;
template <> struct V8<__bf16> { typedef vb8 t; };
template <> struct V8<_Float16> { typedef vh8 t; };
__device__ __forceinline__ f32x16 mfma(vb8 a, vb8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(vh8 a, vh8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float trunc_bf16(float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }
template <class T>
__device__ __forceinline__ void pieces(T v, typename Mat<T>::e out[Mat<T>::P]) {
    if constexpr (Mat<T>::P == 1) out[0] = v;
    else {
        const bool ok = __builtin_isfinite(v);              // an infinity or a NaN travels in the first piece alone
        const float a = ok ? trunc_bf16(v) : v, r = ok ? v - a : 0.0f, b = trunc_bf16(r);
        out[0] = (__bf16)a; out[1] = (__bf16)b; out[2] = (__bf16)(r - b);
    }
}

// ------------------------------------------------------------------------------------------------ one product, any layout
// C[m][n] = sum_k A(m, k) B(n, k):  A(m, k) = a[m lda + k] (AK 1) or a[k lda + m] (AK 0), B likewise.
enum { EPI_OUT = 0, EPI_GATE = 1, EPI_DH = 2 };
struct Prod {
    const void* a; const void* b; int64_t lda, ldb;
    int64_t M, N, K;
    // EPI_OUT: out[m][n] = acc + bias[n] in T, or with `part` the fp32 share of a split over k: part[z][m][n]
    void* out; const void* bias; float* part; int64_t k_per_split;
    // EPI_GATE: N = H; B rows n (gate) and H + n (up); out = h [M][H], bias = b12, p / q fp32 or null.  EPI_DH: out = [dg | du] [M][2H]
    float* p; float* q; int act;
};

// 128 x 128 tiles, 32 deep, four waves of 64 x 64, tiles staged through registers element by element with bounds checks
template <class T, int AK, int BK, int EPI>
__global__ void __launch_bounds__(256) k_ffn_product(Prod g, int tiles_n) {
    typedef typename Mat<T>::e E;
    typedef typename V8<E>::t E8;
    constexpr int P = Mat<T>::P, LD = 40;
    __shared__ __attribute__((aligned(16))) E sA[P][128][LD], sB[P][128][LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 31, lh = lane >> 5;
    const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
    const int64_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    constexpr int NT = EPI == EPI_GATE ? 64 : 128;             // columns of C a tile covers (a gate tile: 64 gate + 64 up)
    const int64_t m0 = tm * 128, n0 = tn * NT;
    const int64_t k_lo = blockIdx.y * g.k_per_split, k_hi = min(g.K, k_lo + g.k_per_split);
    const T* const A = reinterpret_cast<const T*>(g.a);
    const T* const B = reinterpret_cast<const T*>(g.b);
    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;
    // column n of C that row r of the B tile holds, and whether it is an up row
    auto b_row = [&](int r, int64_t& n) -> int64_t {
        if (EPI != EPI_GATE) { n = n0 + r; return n; }
        n = n0 + (r >> 6) * 32 + (r & 31);
        return n + ((r >> 5) & 1) * g.N;
    };
    for (int64_t k0 = k_lo; k0 < k_hi; k0 += 32) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            E e[P];
            {
                const int r = AK ? (tid >> 5) + 8 * i : tid & 127, k = AK ? tid & 31 : (tid >> 7) + 2 * i;
                const int64_t m = m0 + r, kk = k0 + k;
                T v = (T)0.0f;
                if (m < g.M && kk < k_hi) v = A[AK ? m * g.lda + kk : kk * g.lda + m];
                pieces<T>(v, e);
#pragma unroll
                for (int p = 0; p < P; ++p) sA[p][r][k] = e[p];
            }
            {
                const int r = BK ? (tid >> 5) + 8 * i : tid & 127, k = BK ? tid & 31 : (tid >> 7) + 2 * i;
                int64_t n;
                const int64_t row = b_row(r, n), kk = k0 + k;
                T v = (T)0.0f;
                if (n < g.N && kk < k_hi) v = B[BK ? row * g.ldb + kk : kk * g.ldb + row];
                pieces<T>(v, e);
#pragma unroll
                for (int p = 0; p < P; ++p) sB[p][r][k] = e[p];
            }
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            E8 fa[P][2], fb[P][2];
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    fa[p][j] = *reinterpret_cast<const E8*>(&sA[p][wm + 32 * j + lr][16 * ks + 8 * lh]);
                    fb[p][j] = *reinterpret_cast<const E8*>(&sB[p][wn + 32 * j + lr][16 * ks + 8 * lh]);
                }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    if constexpr (P == 3) {
                        acc[a][b] = mfma(fb[2][a], fa[0][b], acc[a][b]);
                        acc[a][b] = mfma(fb[0][a], fa[2][b], acc[a][b]);
                        acc[a][b] = mfma(fb[1][a], fa[1][b], acc[a][b]);
                        acc[a][b] = mfma(fb[1][a], fa[0][b], acc[a][b]);
                        acc[a][b] = mfma(fb[0][a], fa[1][b], acc[a][b]);
                    }
                    acc[a][b] = mfma(fb[0][a], fa[0][b], acc[a][b]);
                }
        }
    }
    // a lane holds row m = lr of C and columns (reg & 3) + 8 (reg >> 2) + 4 lh of each 32 x 32 block
    const T* const bias = reinterpret_cast<const T*>(g.bias);
    T* const out = reinterpret_cast<T*>(g.out);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int64_t m = m0 + wm + 32 * b + lr;
        if (m >= g.M) continue;
        if constexpr (EPI == EPI_GATE) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t n = n0 + (wn >> 6) * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh;
                if (n >= g.N) continue;
                const float gv = acc[0][b][r] + (bias ? (float)bias[n] : 0.0f), uv = acc[1][b][r] + (bias ? (float)bias[g.N + n] : 0.0f);
                float f, df;
                activation<Mat<T>::P == 3>(g.act, gv, f, df);
                out[m * g.N + n] = (T)(f * uv);
                if (g.p) { g.p[m * g.N + n] = uv * df; g.q[m * g.N + n] = f; }
            }
        } else {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int64_t n = n0 + wn + 32 * a + (r & 3) + 8 * (r >> 2) + 4 * lh;
                    if (n >= g.N) continue;
                    const float v = acc[a][b][r];
                    if constexpr (EPI == EPI_DH) {
                        out[m * 2 * g.N + n] = (T)(v * g.p[m * g.N + n]);
                        out[m * 2 * g.N + g.N + n] = (T)(v * g.q[m * g.N + n]);
                    } else if (g.part) g.part[(blockIdx.y * g.M + m) * g.N + n] = v;
                    else out[m * g.N + n] = (T)(v + (bias ? (float)bias[n] : 0.0f));
                }
        }
    }
}

// out[i] = sum_z part[z][i] in increasing z
template <class T>
__global__ void __launch_bounds__(256) k_ffn_join(const float* __restrict__ part, int Z, int64_t n, T* __restrict__ out) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float v = part[i];
        for (int z = 1; z < Z; ++z) v += part[z * n + i];
        out[i] = (T)v;
    }
}

// column sums of a [M][N] matrix: part[y][n] over the rows y, y + gridDim.y, ...; k_ffn_join adds the shares
template <class T>
__global__ void __launch_bounds__(256) k_ffn_colsum(const T* __restrict__ a, int64_t M, int64_t N, float* __restrict__ part) {
    const int64_t n = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (n >= N) return;
    float v = 0.0f;
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) v += (float)a[m * N + n];
    part[blockIdx.y * N + n] = v;
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int CSUM = 64;                                         // shares of a column sum

// shares of a product's k loop when its tiles alone do not fill the chip; each at least 256 deep
inline int k_splits(int64_t M, int64_t N, int64_t K) {
    const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
    return (int)std::max<int64_t>(1, std::min<int64_t>({512 / std::max<int64_t>(tiles, 1), (K + 255) / 256, 64}));
}

template <class T, int AK, int BK, int EPI>
hipError_t product(Prod g, int splits, hipStream_t s) {
    const int nt = EPI == EPI_GATE ? 64 : 128;
    const int64_t tn = (g.N + nt - 1) / nt, tm = (g.M + 127) / 128;
    if (!tm || !tn) return hipSuccess;
    g.k_per_split = splits > 1 ? ((g.K + splits - 1) / splits + 31) / 32 * 32 : std::max<int64_t>(g.K, 1);
    k_ffn_product<T, AK, BK, EPI><<<dim3((unsigned)(tm * tn), splits), 256, 0, s>>>(g, (int)tn);
    return hipGetLastError();
}
template <class T, int AK, int BK>
hipError_t product_split(Prod g, float* part, hipStream_t s) {
    const int z = k_splits(g.M, g.N, g.K);
    if (z == 1) return product<T, AK, BK, EPI_OUT>(g, 1, s);
    g.part = part;
    hipError_t e = product<T, AK, BK, EPI_OUT>(g, z, s);
    if (e != hipSuccess) return e;
    const int64_t n = g.M * g.N;
    k_ffn_join<T><<<(int)std::min<int64_t>((n + 255) / 256, 4096), 256, 0, s>>>(part, z, n, (T*)g.out);
    return hipGetLastError();
}
template <class T>
hipError_t colsum(const void* a, int64_t M, int64_t N, float* part, void* out, hipStream_t s) {
    k_ffn_colsum<T><<<dim3((unsigned)((N + 255) / 256), CSUM), 256, 0, s>>>((const T*)a, M, N, part);
    k_ffn_join<T><<<(int)((N + 255) / 256), 256, 0, s>>>(part, CSUM, N, (T*)out);
    return hipGetLastError();
}

template <class T>
hipError_t forward(const FfnArgs& f, void* ws, hipStream_t s) {
    Prod g{};
    g.a = f.x; g.lda = f.D; g.b = f.w12; g.ldb = f.D; g.M = f.M; g.N = f.H; g.K = f.D;
    g.out = f.h ? f.h : ws; g.bias = f.b12; g.act = f.act;
    if (f.pq) { g.p = f.pq; g.q = f.pq + f.M * f.H; }
    hipError_t e = product<T, 1, 1, EPI_GATE>(g, 1, s);
    if (e != hipSuccess) return e;
    Prod d{};
    d.a = g.out; d.lda = f.H; d.b = f.w3; d.ldb = f.H; d.M = f.M; d.N = f.O; d.K = f.H; d.out = f.y; d.bias = f.b3;
    return product<T, 1, 1, EPI_OUT>(d, 1, s);
}

template <class T>
hipError_t backward(const FfnArgs& f, void* ws, hipStream_t s) {
    T* const dgu = reinterpret_cast<T*>(ws);
    float* const part = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + ((size_t)f.M * 2 * f.H * sizeof(T) + 255) / 256 * 256);
    hipError_t e = hipSuccess;
    if (f.dx || f.dw12 || f.db12) {
        Prod g{};
        g.a = f.dy; g.lda = f.O; g.b = f.w3; g.ldb = f.H; g.M = f.M; g.N = f.H; g.K = f.O; g.out = dgu; g.p = f.pq; g.q = f.pq + f.M * f.H;
        if ((e = product<T, 1, 0, EPI_DH>(g, 1, s)) != hipSuccess) return e;
    }
    if (f.dx) {
        Prod g{};
        g.a = dgu; g.lda = 2 * (int64_t)f.H; g.b = f.w12; g.ldb = f.D; g.M = f.M; g.N = f.D; g.K = 2 * (int64_t)f.H; g.out = f.dx;
        if ((e = product<T, 1, 0, EPI_OUT>(g, 1, s)) != hipSuccess) return e;
    }
    if (f.dw12) {
        Prod g{};
        g.a = dgu; g.lda = 2 * (int64_t)f.H; g.b = f.x; g.ldb = f.D; g.M = 2 * (int64_t)f.H; g.N = f.D; g.K = f.M; g.out = f.dw12;
        if ((e = product_split<T, 0, 0>(g, part, s)) != hipSuccess) return e;
    }
    if (f.dw3) {
        Prod g{};
        g.a = f.dy; g.lda = f.O; g.b = f.h; g.ldb = f.H; g.M = f.O; g.N = f.H; g.K = f.M; g.out = f.dw3;
        if ((e = product_split<T, 0, 0>(g, part, s)) != hipSuccess) return e;
    }
    if (f.db12 && (e = colsum<T>(dgu, f.M, 2 * (int64_t)f.H, part, f.db12, s)) != hipSuccess) return e;
    if (f.db3 && (e = colsum<T>(f.dy, f.M, f.O, part, f.db3, s)) != hipSuccess) return e;
    return hipSuccess;
}

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

size_t ffn_forward_workspace(const FfnArgs& a, bool keeps_h) { return keeps_h ? 0 : up256((size_t)a.M * a.H * dt_size(a.dt)); }

size_t ffn_backward_workspace(const FfnArgs& a) {
    size_t part = std::max((size_t)CSUM * 2 * a.H * 4, (size_t)CSUM * a.O * 4);
    const auto split = [&](int64_t M, int64_t N) {
        const int z = k_splits(M, N, a.M);
        if (z > 1) part = std::max(part, (size_t)z * M * N * 4);
    };
    split(2 * (int64_t)a.H, a.D);
    split(a.O, a.H);
    return up256((size_t)a.M * 2 * a.H * dt_size(a.dt)) + up256(part);
}

hipError_t launch_ffn_forward(const FfnArgs& a, void* ws, hipStream_t s) {
    return a.dt == IFF_DT_F32 ? forward<float>(a, ws, s) : a.dt == IFF_DT_BF16 ? forward<__bf16>(a, ws, s) : forward<_Float16>(a, ws, s);
}
hipError_t launch_ffn_backward(const FfnArgs& a, void* ws, hipStream_t s) {
    return a.dt == IFF_DT_F32 ? backward<float>(a, ws, s) : a.dt == IFF_DT_BF16 ? backward<__bf16>(a, ws, s) : backward<_Float16>(a, ws, s);
}
